"""8-bit blocks, Linear on them, weight gradients and GeGLU from 8-bit checkpoints, LayerNorm forward / backward: every
operator against a plain implementation in 64 bits.

Tolerances come from the arithmetic: U = 2^-24 is half a step of f32, 2^-8 of bf16.  A sum of n f32 terms in any order is
off by at most (n - 1) U times the sum of the terms' magnitudes; the 8-bit values themselves, and whatever is exact by
construction, have to be equal bit for bit.
"""
import math

import numpy as np
import pytest
import torch

import sd_amd  # noqa: F401
from sd_amd import _lib, ops

pytestmark = pytest.mark.gpu
torch.set_grad_enabled(False)
DEV = "cuda"
U, UB = 2.0 ** -24, 2.0 ** -8
F32, BF16, E4M3, E5M2 = torch.float32, torch.bfloat16, torch.float8_e4m3fn, torch.float8_e5m2


def gen(seed):
    return torch.Generator().manual_seed(seed)


def rnd(seed, shape, dtype=F32, scale=1.0):
    """Rows and columns of uneven size, as hidden states have."""
    g = gen(seed)
    x = torch.randn(shape, generator=g) * scale
    if len(shape) == 2:
        x = x * torch.exp(0.5 * torch.randn(shape[1], generator=g)) * torch.exp(0.3 * torch.randn(shape[0], 1, generator=g))
    return x.to(dtype)


# ------------------------------------------------------------------ the plain forms, 64 bits
def grid8(v, fmt):
    """Nearest value of the 8-bit type, ties to even, for |v| within its range (float64 in and out)."""
    bits, low = (3, -6) if fmt == E4M3 else (2, -14)
    m, e = np.frexp(np.abs(v))                       # |v| = m 2^e, m in [0.5, 1)
    step = np.ldexp(1.0, np.maximum(e - 1, low) - bits)
    return np.copysign(np.rint(np.abs(v) / step) * step, v)


def blocks_ref(x, fmt, block_rows=1):
    """(values, scale exponents [rows / block_rows, KB]) of x [rows, K] (float64)."""
    rows, K = x.shape
    kb, rb = -(-K // 128), -(-rows // block_rows)
    top = 448.0 if fmt == E4M3 else 57344.0
    out, exps = np.zeros_like(x), np.zeros((rb, kb), dtype=np.int64)
    for b in range(kb):
        for r in range(rb):
            rs, cs = slice(r * block_rows, (r + 1) * block_rows), slice(b * 128, (b + 1) * 128)
            part = x[rs, cs]
            fin = np.abs(part[np.isfinite(part)])
            amax = fin.max() if fin.size else 0.0
            e = 0
            if amax > 0:
                e = math.frexp(amax / top)[1]        # top * 2^(e-1) < amax up to the quotient's rounding: settled below
                while top * 2.0 ** (e - 1) >= amax:
                    e -= 1
                while top * 2.0 ** e < amax:
                    e += 1
                e = max(e, -126)
            exps[r, b] = e
            with np.errstate(invalid="ignore"):
                q = grid8(np.where(np.isfinite(part), part, 0) * 2.0 ** -e, fmt) * 2.0 ** e
            keep = np.isinf(part) if fmt == E5M2 else np.zeros(part.shape, bool)
            q = np.where(np.isnan(part) | (np.isinf(part) & ~keep), np.nan, np.where(keep, part, q))
            out[rs, cs] = q
    return out, exps


def np64(t):
    return t.detach().float().cpu().numpy().astype(np.float64)


def scales_of(b):
    kb = -(-b.shape[-1] // 128)
    s = b.scale.cpu().numpy().astype(np.int64)
    assert (s[:, kb:] == 127).all()                  # the padding up to whole words
    return s[:, :kb] - 127


def close(got, want, tol, what=""):
    """Elementwise |got - want| <= tol."""
    got = got if isinstance(got, np.ndarray) else np64(got)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.size} off, worst {np.max(np.abs(got - want) / np.maximum(tol, 1e-300)):.3g} x tolerance"


# ------------------------------------------------------------------ blocks
@pytest.mark.parametrize("rows,K", [(1, 1), (3, 7), (2, 128), (5, 129), (77, 320), (33, 1001), (4, 127), (300, 640)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("fmt", [E4M3, E5M2])
def test_quantize8_is_exact(rows, K, dtype, fmt):
    x = rnd(rows * 7 + K, (rows, K), dtype)
    b = ops.quantize8(x.to(DEV), fmt)
    want, exps = blocks_ref(np64(x), fmt)
    assert np.array_equal(scales_of(b), exps)
    for out in (F32, BF16):
        assert np.array_equal(np64(b.dequantize(out)), want)
    assert (b.q.view(torch.uint8)[:, K:] == 0).all()
    assert b.shape == (rows, K) and b.dtype == fmt and b.nbytes == b.q.numel() + b.scale.numel()


def test_quantize8_borders():
    """Maxima next to the border between two scales, ties, zeros, tiny and huge blocks, NaN and infinities."""
    x = torch.zeros(12, 128)
    x[0, 5] = 448.0
    x[1, 5] = np.nextafter(np.float32(448), np.float32(500)).item()
    x[2] = torch.arange(128) * 3.5 + 0.25
    x[3, 0], x[3, 1] = 448.0, 17.0                   # 17 ties between 16 and 18
    x[4, 0], x[4, 1], x[4, 2] = 448.0, 2.0 ** -10, 3 * 2.0 ** -10   # half of the smallest step, one and a half
    x[5] = 1e-41                                     # subnormal
    x[6, 3] = 3.0e38
    x[7, 0], x[7, 1], x[7, 2] = float("inf"), -float("inf"), 2.5
    x[8, 0], x[8, 1] = float("nan"), -1.5
    x[9] = float("nan")
    x[10] = -0.0
    x[11, 64] = -57344.0 * 2.0 ** 60
    for fmt in (E4M3, E5M2):
        b = ops.quantize8(x.to(DEV), fmt)
        want, exps = blocks_ref(np64(x), fmt)
        assert np.array_equal(scales_of(b), exps)
        got = np64(b.dequantize(F32))
        assert np.array_equal(got, want, equal_nan=True)


def test_quantize8_takes_row_strides_and_refuses_others():
    base = rnd(5, (9, 400)).to(DEV)
    got = ops.quantize8(base[:, 3:203])
    assert np.array_equal(np64(got.dequantize(F32)), blocks_ref(np64(base[:, 3:203].cpu()), E4M3)[0])
    same = ops.quantize8(base[:1].expand(4, 400))
    assert np.array_equal(np64(same.dequantize(F32)), np.repeat(blocks_ref(np64(base[:1].cpu()), E4M3)[0], 4, 0))
    with pytest.raises(_lib.SdamdError):
        ops.quantize8(base.t())
    with pytest.raises(TypeError):
        ops.quantize8(base, torch.int8)
    with pytest.raises(TypeError):
        ops.quantize8(base.half())
    empty = ops.quantize8(torch.empty(0, 320, device=DEV))
    assert empty.shape == (0, 320) and empty.dequantize().shape == (0, 320)


@pytest.mark.parametrize("N,K", [(1, 1), (5, 300), (128, 128), (129, 127), (333, 215), (640, 320)])
@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize8_weight_is_exact(N, K, dtype):
    w = rnd(N + K, (N, K), dtype)
    want, exps = blocks_ref(np64(w), E4M3, 128)
    b = ops.quantize8_weight(w.to(DEV))
    assert np.array_equal(scales_of(b), exps) and np.array_equal(np64(b.dequantize(F32)), want)
    t = ops.quantize8_weight(w.to(DEV).t())          # the transposed weight: any strides
    assert t.shape == (K, N) and np.array_equal(np64(t.dequantize(BF16)), want.T)
    assert (b.q.view(torch.uint8)[:, K:] == 0).all()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_quantize8_weight_takes_any_strides(dtype):
    big = rnd(3, (300, 700), dtype)
    big[7, 20], big[140, 300] = float("nan"), float("inf")
    dev = big.to(DEV)
    views = [lambda t: t[5:205, 3:604], lambda t: t[::2, ::3], lambda t: t[5:205, 3:604].t(), lambda t: t[::3, 1:300:2].t(),
             lambda t: t[4:5, 9:400].expand(150, 391), lambda t: t[9:200, 4:5].expand(191, 140), lambda t: t[3:100, 5:10], lambda t: t[3:8, :300:7]]
    for view in views:
        a, b = ops.quantize8_weight(view(dev)), ops.quantize8_weight(view(dev).contiguous())
        assert torch.equal(a.q.view(torch.uint8), b.q.view(torch.uint8)) and torch.equal(a.scale, b.scale)
        plain = torch.where(view(big).isfinite(), view(big), torch.zeros((), dtype=dtype))
        want, exps = blocks_ref(np64(plain), E4M3, 128)
        assert np.array_equal(scales_of(a), exps)
        got, fin = np64(a.dequantize(F32)), view(big).isfinite().numpy()
        assert np.array_equal(got[fin], want[fin]) and np.isnan(got[~fin]).all()


# ------------------------------------------------------------------ Linear
def linear_ref(xq, wq, bias, res, act):
    v = xq @ wq.T
    mag = np.abs(xq) @ np.abs(wq).T
    for t in (bias, res):
        if t is not None:
            v, mag = v + np64(t), mag + np.abs(np64(t))
    if act == ops.ACT_SILU:
        v = v / (1 + np.exp(-v))
    elif act == ops.ACT_QUICK_GELU:
        v = v / (1 + np.exp(-1.702 * v))
    return v, mag


def linear_tol(xq, wq, mag, out, want, act):
    K = xq.shape[1]
    if out == F32:
        tol = (K + 4) * U * mag
    else:
        # inside an 8-bit instruction 128 products are cut 2^-18 below the largest at the coarsest: 128 * 2^-18 of it per
        # block; then f32 sums over the blocks and one rounding to bf16
        kb = -(-K // 128)
        cut = np.zeros_like(mag)
        for b in range(kb):
            c = slice(b * 128, b * 128 + 128)
            cut += np.outer(np.abs(xq[:, c]).max(1), np.abs(wq[:, c]).max(1)) * 2.0 ** -11
        tol = cut + (kb + 4) * U * mag + UB * np.abs(want)
    if act:                                          # slope at most 1.1, and 8 roundings in the activation itself
        tol = 1.1 * tol + 8 * U * np.abs(want)
    return tol


SHAPES = [(1, 320, 1280), (1, 5, 3), (2, 129, 17), (16, 640, 40), (17, 320, 320), (33, 1001, 130), (64, 768, 640),
          (154, 768, 640), (200, 300, 333), (1100, 640, 1500), (1500, 257, 2050)]


@pytest.mark.parametrize("M,K,N", SHAPES)
@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("fmt", [E4M3, E5M2])
def test_linear8(M, K, N, out, fmt):
    x = rnd(M + K, (M, K), BF16 if N % 2 else F32)
    w = rnd(N + K, (N, K), scale=K ** -0.5)
    bias = rnd(1, (N,)) if (M + N) % 2 else None
    res = rnd(2, (M, N), out) if N % 3 else None
    act = [ops.ACT_NONE, ops.ACT_SILU, ops.ACT_QUICK_GELU][(M + K + N) % 3]
    xq, wq = blocks_ref(np64(x), fmt)[0], blocks_ref(np64(w), E4M3, 128)[0]
    want, mag = linear_ref(xq, wq, bias, res, act)
    tol = linear_tol(xq, wq, mag, out, want, act)
    wb = ops.quantize8_weight(w.to(DEV))
    dev = [None if t is None else t.to(DEV) for t in (bias, res)]
    got = ops.linear8(x.to(DEV), wb, dev[0], dev[1], act, out, fmt)
    assert got.dtype == out and got.shape == (M, N)
    close(got, want, tol, "rows given")
    again = ops.linear8(ops.quantize8(x.to(DEV), fmt), wb, dev[0], dev[1], act, out)
    assert torch.equal(got, again)                   # quantised ahead of time or on the way: the same bits
    if N % 7 and N > 3:
        rel = np.linalg.norm(np64(got) - want) / max(np.linalg.norm(want), 1e-30)
        assert rel < (UB if out == BF16 else 1e-5)


@pytest.mark.parametrize("out", [BF16, F32])
def test_linear8_large_tile(out):
    """Enough tiles for the 256 x 256 form (bf16), with ragged edges in every direction; checked on rows and columns."""
    M, K, N = 4100, 450, 3500
    x, w = rnd(3, (M, K), BF16), rnd(4, (N, K), scale=K ** -0.5)
    got = np64(ops.linear8(x.to(DEV), ops.quantize8_weight(w.to(DEV)), out_dtype=out))
    xq, wq = blocks_ref(np64(x), E4M3)[0], blocks_ref(np64(w), E4M3, 128)[0]
    want = xq @ wq.T
    close(got, want, linear_tol(xq, wq, np.abs(xq) @ np.abs(wq).T, out, want, 0), "large")


@pytest.mark.parametrize("M,K,N", [(256, 640, 640), (1000, 200, 640), (1500, 257, 2050), (2048, 130, 2304), (4100, 260, 3501), (4096, 128, 4096)])
@pytest.mark.parametrize("out", [BF16, F32])
def test_linear8_epilogues_of_every_kernel(M, K, N, out):
    """Bias, residual and activation together at sizes that reach each kernel, with whole tiles and ragged ones; the residual
    may be the output."""
    x, w = rnd(3, (M, K), BF16), rnd(4, (N, K), scale=K ** -0.5)
    bias, res = rnd(5, (N,)), rnd(6, (M, N), out)
    xq, wq = blocks_ref(np64(x), E4M3)[0], blocks_ref(np64(w), E4M3, 128)[0]
    wb, bd = ops.quantize8_weight(w.to(DEV)), bias.to(DEV)
    for b, r, act in ((bias, res, ops.ACT_SILU), (None, res, ops.ACT_NONE), (bias, None, ops.ACT_NONE), (None, None, ops.ACT_QUICK_GELU)):
        want, mag = linear_ref(xq, wq, b, r, act)
        io = None if r is None else r.to(DEV)
        got = ops.linear8(x.to(DEV), wb, None if b is None else bd, io, act, out, out=io)
        close(got, want, linear_tol(xq, wq, mag, out, want, act), f"bias {b is not None} residual {r is not None} act {act}")


def test_linear8_planned_batch_of_many_samples():
    """Few rows a sample, more in all than one launch of the rows kernel takes."""
    S, R, K, N = 131100, 8, 8, 16
    x, w = rnd(3, (S * R, K)).to(DEV), ops.quantize8_weight(rnd(4, (N, K)).to(DEV))
    res = rnd(5, (S * R, N)).to(DEV)
    with ops.plan_samples(S):
        for xx in (x, ops.quantize8(x)):
            batch = ops.linear8(xx, w, residual=res)
            for s in (0, 131070, 131099):
                rows = slice(s * R, s * R + R)
                with ops.plan_samples(1):
                    alone = ops.linear8(x[rows], w, residual=res[rows])
                assert torch.equal(batch[rows], alone)


def test_linear8_scale_range():
    """Blocks of very different size in one row, tiny ones and huge ones: the scales do the work."""
    M, K, N = 40, 640, 96
    for out in (BF16, F32):
        x = rnd(6, (M, K)) * torch.exp2(torch.arange(K).div(128, rounding_mode="floor") * 12.0 - 30)
        w = rnd(7, (N, K)) * torch.exp2(20 - torch.arange(K).div(128, rounding_mode="floor") * 11.0)
        xq, wq = blocks_ref(np64(x), E4M3)[0], blocks_ref(np64(w), E4M3, 128)[0]
        want, mag = linear_ref(xq, wq, None, None, 0)
        got = ops.linear8(x.to(DEV), ops.quantize8_weight(w.to(DEV)), out_dtype=out)
        close(got, want, linear_tol(xq, wq, mag, out, want, 0))


@pytest.mark.parametrize("M", [3, 40, 300])
@pytest.mark.parametrize("out", [BF16, F32])
def test_linear8_keeps_nan_in_its_row(M, out):
    K, N = 300, 260
    x, w = rnd(8, (M, K)), rnd(9, (N, K))
    x[1, 299] = float("nan")
    x[2, 0] = float("inf")
    clean = x.clone()
    clean[1], clean[2] = 0, 0
    wb = ops.quantize8_weight(w.to(DEV))
    got, ref = ops.linear8(x.to(DEV), wb, out_dtype=out).cpu(), ops.linear8(clean.to(DEV), wb, out_dtype=out).cpu()
    assert got[1].isnan().all() and got[2].isnan().all()
    rest = [i for i in range(M) if i not in (1, 2)]
    assert torch.equal(got[rest], ref[rest])


def test_linear8_shapes_out_and_refusals():
    w = ops.quantize8_weight(rnd(1, (48, 200)).to(DEV))
    x = rnd(2, (2, 5, 200), BF16).to(DEV)
    y = ops.linear8(x, w)
    assert y.shape == (2, 5, 48) and y.dtype == BF16
    buf = torch.empty(2, 5, 48, dtype=BF16, device=DEV)
    assert ops.linear8(x, w, out=buf) is buf and torch.equal(buf, y)
    assert ops.linear8(x[0, 0], w).shape == (48,)
    strided = torch.zeros(40, 230, device=DEV)
    strided[:, 7:207] = rnd(3, (40, 200)).to(DEV)
    assert torch.equal(ops.linear8(strided[:, 7:207], w), ops.linear8(strided[:, 7:207].contiguous(), w))
    assert torch.equal(ops.linear8(strided[:4, 7:207], w), ops.linear8(strided[:4, 7:207].contiguous(), w))
    assert ops.linear8(torch.empty(0, 200, device=DEV), w).shape == (0, 48)
    square = torch.zeros(64, 64, device=DEV)
    bad = [lambda: ops.linear8(x, x), lambda: ops.linear8(x[..., :100], w), lambda: ops.linear8(x, w, bias=torch.zeros(47, device=DEV)),
           lambda: ops.linear8(x, w, bias=torch.zeros(48, device=DEV, dtype=BF16)),
           lambda: ops.linear8(x, w, residual=torch.zeros(2, 5, 48, device=DEV), out_dtype=BF16),
           lambda: ops.linear8(x, w, act=ops.ACT_GEGLU), lambda: ops.linear8(x, w, out=buf[:1]), lambda: ops.linear8(w, w),
           lambda: ops.linear8(square, ops.quantize8_weight(square), out=square),
           lambda: ops.linear8(x.cpu(), w)]
    for call in bad:
        with pytest.raises(_lib.SdamdError):
            call()
    for call in (lambda: ops.linear8(x, w, out_dtype=torch.float16), lambda: ops.linear8(x.half(), w), lambda: ops.linear8(x, w, fmt=BF16)):
        with pytest.raises(TypeError):
            call()


def test_scale_bytes_of_any_value():
    """Blocks made elsewhere may carry any scale byte: 2^-127 (0) to 2^127 (254), and 255, which stands for NaN."""
    M, K, N = 40, 256, 130
    x = ops.quantize8((rnd(1, (M, K)).sign() * 256).to(DEV))
    w = ops.quantize8_weight(rnd(2, (N, K)).to(DEV))
    bytes_ = [0, 1, 60, 127, 200, 254, 255, 130]
    for r in range(M):
        x.scale[r, :2] = bytes_[r % len(bytes_)]
    w.scale[:, :2] = 70                                  # 2^-57
    vals = np64(x.q) * np.repeat(2.0 ** (x.scale[:, :2].cpu().numpy().astype(np.float64) - 127), 128, 1)
    nan = x.scale[:, 0].cpu().numpy() == 255
    wv = np64(w.q) * 2.0 ** -57
    want = vals @ wv.T
    top = np.finfo(np.float32).max
    # 2^127 * 256 is beyond float32 (and bfloat16, of the same range): where values are taken in those types, such a one is an
    # infinity, like in any conversion.  The bfloat16 form of the product takes the bytes themselves.
    with np.errstate(over="ignore"):
        held = vals.astype(np.float32).astype(np.float64)
    for out in (BF16, F32):
        for rows in (slice(0, 8), slice(0, M)):
            part = ops.Blocks8(x.q[rows].contiguous(), x.scale[rows].contiguous(), (len(range(*rows.indices(M))), K))
            got = np64(ops.linear8(part, w, out_dtype=out))
            assert np.isnan(got[nan[rows]]).all()
            ok = ~nan[rows] & (np.isfinite(held[rows]).all(1) if out == F32 else True)
            assert not np.isfinite(got[~ok]).any() and (np.abs(want[rows][ok]) < top).all()
            # scale byte 0 puts results at 2^-127 2^8 2^-57 2^8 sqrt(256) = 2^-164, below everything an f32 or bf16 holds: such
            # a result is off by itself, less than the smallest normal number 2^-126
            close(got[ok], want[rows][ok], 2.0 ** -126 + linear_tol(vals[rows][ok], wv, np.abs(vals[rows][ok]) @ np.abs(wv).T, out, want[rows][ok], 0))
    assert np.isnan(np64(x.dequantize(F32))[nan]).all() and np.array_equal(np64(x.dequantize(F32))[~nan], held[~nan])
    dy = torch.zeros(M, 24, dtype=BF16)
    dy[4:6] = 2.0 ** -60                                 # scales 2^73 and 2^127
    dw, _ = ops.linear8_weight_grad(dy[4:6].contiguous().to(DEV), ops.Blocks8(x.q[4:6].contiguous(), x.scale[4:6].contiguous(), (2, K)))
    assert np.isinf(held[5]).all() and np.array_equal(np64(dw), np64(dy[4:6]).T @ held[4:6])
    dw, _ = ops.linear8_weight_grad(dy[6:7].contiguous().to(DEV), ops.Blocks8(x.q[6:7].contiguous(), x.scale[6:7].contiguous(), (1, K)))
    assert dw.isnan().all()


@pytest.mark.parametrize("out", [BF16, F32])
def test_linear8_under_plan_samples(out):
    """Deterministic plans: a sample's rows give the same bits alone and in any batch."""
    S, R, K, N = 24, 77, 320, 640
    x, w = rnd(3, (S * R, K)).to(DEV), ops.quantize8_weight(rnd(4, (N, K)).to(DEV))
    with ops.plan_samples(1):
        alone = ops.linear8(x[5 * R:6 * R], w, out_dtype=out)
    with ops.plan_samples(S):
        batch = ops.linear8(x, w, out_dtype=out)
    assert torch.equal(batch[5 * R:6 * R], alone)


# ------------------------------------------------------------------ weight gradient
@pytest.mark.parametrize("T,N,K", [(1, 1, 1), (3, 8, 130), (64, 16, 128), (77, 40, 300), (1003, 333, 215), (130, 1280, 320),
                                   (4100, 264, 257), (700, 2100, 1100), (640, 2056, 1024), (70, 5, 200), (300, 7, 129), (65, 3, 1300), (129, 9, 64),
                                   (100, 12, 300), (1500, 2563, 2100), (5000, 4098, 1024)])
@pytest.mark.parametrize("fmt", [E4M3, E5M2])
def test_weight_grad(T, N, K, fmt):
    x, dy = rnd(T + K, (T, K)), rnd(T + N, (T, N), BF16, 0.1)
    xq, d = blocks_ref(np64(x), fmt)[0], np64(dy)
    x8 = ops.quantize8(x.to(DEV), fmt)
    dw, db = ops.linear8_weight_grad(dy.to(DEV), x8)
    assert dw.dtype == F32 and db.dtype == F32
    # products of two 8-bit-exponent bf16 values are exact in f32
    close(dw, d.T @ xq, (T + 2) * U * (np.abs(d).T @ np.abs(xq)), "dw")
    close(db, d.sum(0), (T + 2) * U * np.abs(d).sum(0), "db")
    dw2, none = ops.linear8_weight_grad(dy.to(DEV), x8, bias=False)
    assert none is None and torch.equal(dw2, dw)     # the same bits every run


def test_weight_grad_misaligned_and_nan():
    T, N, K = 100, 64, 140
    buf = torch.zeros(T * N + 1, dtype=BF16, device=DEV)
    dy = buf[1:].view(T, N)
    dy.copy_(rnd(1, (T, N), BF16).to(DEV))
    x = rnd(2, (T, K))
    x[5, 3] = float("nan")
    x8 = ops.quantize8(x.to(DEV))
    dw, db = ops.linear8_weight_grad(dy, x8)
    dw2, db2 = ops.linear8_weight_grad(dy.clone(), x8)
    assert torch.equal(dw.nan_to_num(7.0), dw2.nan_to_num(7.0)) and torch.equal(db, db2)
    assert dw[:, 3].isnan().all() and not dw[:, :3].isnan().any() and not dw[:, 4:].isnan().any()
    with pytest.raises(TypeError):
        ops.linear8_weight_grad(dy.float(), x8)
    for bad in (lambda: ops.linear8_weight_grad(dy[:50], x8), lambda: ops.linear8_weight_grad(dy, x.to(DEV)),
                lambda: ops.linear8_weight_grad(dy[:, ::2], x8)):
        with pytest.raises(_lib.SdamdError):
            bad()
    zw, zb = ops.linear8_weight_grad(torch.empty(0, 9, dtype=BF16, device=DEV), ops.quantize8(torch.empty(0, 33, device=DEV)))
    assert zw.shape == (9, 33) and not zw.any() and zb.shape == (9,) and not zb.any()


# ------------------------------------------------------------------ LayerNorm
WIDTHS = [1, 3, 8, 77, 128, 320, 384, 500, 640, 768, 1001, 1024, 1280, 1536, 2048, 2560, 4096, 5120, 12288]


def norm_ref(x, gamma, beta, eps):
    mean = x.mean(1, keepdims=True)
    rstd = 1 / np.sqrt(((x - mean) ** 2).mean(1, keepdims=True) + eps)
    xh = (x - mean) * rstd
    # a sum over a row is at most 48 values after one another, 8 shuffle steps and 3 adds
    e_mean = 64 * U * np.abs(x).mean(1, keepdims=True)
    e_xh = e_mean * rstd + 80 * U * np.abs(xh) + 2 * U
    return mean, rstd, xh, xh * gamma + beta, e_mean, e_xh


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("dtype,out", [(F32, F32), (F32, BF16), (BF16, BF16), (BF16, F32)])
def test_layernorm_train(C, dtype, out):
    rows = 37 if C < 2000 else 6
    x = (rnd(C, (rows, C)) + 3.0).to(dtype)
    gamma, beta = 1 + 0.2 * rnd(1, (C,)), 0.2 * rnd(2, (C,))
    y, mean, rstd = ops.layernorm_train(x.to(DEV), gamma.to(DEV), beta.to(DEV), 1e-5, out)
    m, r, xh, want, e_mean, e_xh = norm_ref(np64(x), np64(gamma), np64(beta), 1e-5)
    close(mean, m[:, 0], e_mean[:, 0], "mean")
    close(rstd, r[:, 0], 80 * U * r[:, 0], "rstd")
    tol = e_xh * np.abs(np64(gamma)) + 4 * U * (np.abs(want) + np.abs(np64(beta)))
    close(y, want, tol + (UB * np.abs(want) if out == BF16 else 0), "y")
    if C in (320, 1001, 4096):
        for fmt in (E4M3, E5M2):
            yb = ops.layernorm_train(x.to(DEV), gamma.to(DEV), beta.to(DEV), 1e-5, fmt)[0]
            y32 = ops.layernorm_train(x.to(DEV), gamma.to(DEV), beta.to(DEV), 1e-5, F32)[0]
            two = ops.quantize8(y32, fmt)            # in one pass or in two: the same bytes
            assert torch.equal(yb.q.view(torch.uint8), two.q.view(torch.uint8)) and torch.equal(yb.scale, two.scale)


@pytest.mark.parametrize("C", [1, 9, 128, 200, 320, 640, 700, 1280, 3000, 5000])
def test_layernorm_train_blocks(C):
    rows = 19
    x, gamma, beta = rnd(C, (rows, C)).to(DEV), (1 + 0.2 * rnd(1, (C,))).to(DEV), (0.2 * rnd(2, (C,))).to(DEV)
    yb = ops.layernorm_train(x, gamma, beta, 1e-5, E4M3)[0]
    two = ops.quantize8(ops.layernorm_train(x, gamma, beta, 1e-5, F32)[0], E4M3)
    assert torch.equal(yb.q.view(torch.uint8), two.q.view(torch.uint8)) and torch.equal(yb.scale, two.scale)


def backward_ref(dy, x, gamma, res, eps):
    mean, rstd, xh, _, _, e_xh = norm_ref(x, gamma, np.zeros_like(gamma), eps)
    a = dy * gamma
    s1, s2 = a.mean(1, keepdims=True), (a * xh).mean(1, keepdims=True)
    dx = rstd * (a - s1 - xh * s2) + (0 if res is None else res)
    mag = np.abs(a) + np.abs(a).mean(1, keepdims=True) + np.abs(xh) * np.abs(a * xh).mean(1, keepdims=True)
    tol = rstd * (100 * U * mag + e_xh * np.abs(s2) + np.abs(xh) * (np.abs(a) * e_xh).mean(1, keepdims=True))
    tol = tol + 4 * U * (np.abs(dx) + (0 if res is None else np.abs(res)))
    return dx, (dy * xh).sum(0), dy.sum(0), tol, (np.abs(dy) * e_xh).sum(0), np.abs(dy * xh).sum(0)


@pytest.mark.parametrize("C", WIDTHS)
@pytest.mark.parametrize("xt,dt,skip", [(F32, F32, False), (F32, BF16, True), (BF16, BF16, False), (BF16, F32, True), (E4M3, BF16, True), (E5M2, F32, False)])
def test_layernorm_backward(C, xt, dt, skip):
    rows = 1 if C == 77 else 300 if C == 320 else 41 if C < 2000 else 7
    x = rnd(C, (rows, C)) + 0.5
    dy, gamma = rnd(C + 1, (rows, C), dt, 0.1), 1 + 0.2 * rnd(3, (C,))
    if xt in (E4M3, E5M2):
        kept = ops.quantize8(x.to(DEV), xt)
        vals, ot = kept.dequantize(F32), dt
        given = kept
    else:
        given = vals = x.to(xt).to(DEV)
        ot = xt
    res = rnd(9, (rows, C), ot) if skip else None
    _, mean, rstd = ops.layernorm_train(vals, gamma.to(DEV), torch.zeros(C, device=DEV))
    dx, dg, db = ops.layernorm_backward(dy.to(DEV), given, gamma.to(DEV), mean, rstd, None if res is None else res.to(DEV))
    assert dx.dtype == ot
    w_dx, w_dg, w_db, tol, e_g, mag_g = backward_ref(np64(dy), np64(vals), np64(gamma), None if res is None else np64(res), 1e-5)
    close(dx, w_dx, tol + (UB * np.abs(w_dx) if ot == BF16 else 0), "dx")
    close(dg, w_dg, e_g + (rows + 64) * U * mag_g, "dgamma")
    close(db, w_db, (rows + 64) * U * np.abs(np64(dy)).sum(0), "dbeta")
    again = ops.layernorm_backward(dy.to(DEV), given, gamma.to(DEV), mean, rstd, None if res is None else res.to(DEV))
    assert all(torch.equal(a, b) for a, b in zip(again, (dx, dg, db)))


def test_layernorm_backward_many_rows():
    rows, C = 20011, 320
    x, dy = rnd(1, (rows, C)), rnd(2, (rows, C), BF16)
    gamma = 1 + 0.2 * rnd(3, (C,))
    _, mean, rstd = ops.layernorm_train(x.to(DEV), gamma.to(DEV), torch.zeros(C, device=DEV))
    dx, dg, db = ops.layernorm_backward(dy.to(DEV), x.to(DEV), gamma.to(DEV), mean, rstd)
    w_dx, w_dg, w_db, tol, e_g, mag_g = backward_ref(np64(dy), np64(x), np64(gamma), None, 1e-5)
    close(dx, w_dx, tol, "dx")
    # 512 workgroups of 32 rows at a time: 20 rows after one another, 3 shuffles, 4 waves, 512 / 16 + 16 partial rows
    close(dg, w_dg, e_g + 128 * U * mag_g, "dgamma")
    close(db, w_db, 128 * U * np.abs(np64(dy)).sum(0), "dbeta")


def test_layernorm_gradient_against_differences():
    """The kernels' dx, dgamma and dbeta along random directions against central differences of the 64-bit forward pass."""
    rows, C, eps, h = 11, 300, 1e-5, 1e-4
    x, dy = rnd(1, (rows, C)), rnd(2, (rows, C))
    gamma, beta = 1 + 0.2 * rnd(3, (C,)), 0.2 * rnd(4, (C,))
    _, mean, rstd = ops.layernorm_train(x.to(DEV), gamma.to(DEV), beta.to(DEV), eps)
    dx, dg, db = (np64(t) for t in ops.layernorm_backward(dy.to(DEV), x.to(DEV), gamma.to(DEV), mean, rstd))
    X, D, G, B = np64(x), np64(dy), np64(gamma), np64(beta)
    loss = lambda a, g, b: float((norm_ref(a, g, b, eps)[3] * D).sum())  # noqa: E731
    r = np.random.default_rng(0)
    for _ in range(4):
        vx, vg, vb = r.standard_normal((rows, C)), r.standard_normal(C), r.standard_normal(C)
        for got, fd, size in (((dx * vx).sum(), (loss(X + h * vx, G, B) - loss(X - h * vx, G, B)) / (2 * h), np.abs(dx * vx).sum()),
                              ((dg * vg).sum(), (loss(X, G + h * vg, B) - loss(X, G - h * vg, B)) / (2 * h), np.abs(dg * vg).sum()),
                              ((db * vb).sum(), (loss(X, G, B + h * vb) - loss(X, G, B - h * vb)) / (2 * h), np.abs(db * vb).sum())):
            # f32 gradients are off by < 2^-16 of their size (bounds above); the difference by h^2 times the third derivative
            assert abs(got - fd) <= 2.0 ** -16 * size + 1e-5 * abs(fd) + 1e-6


def test_layernorm_refusals_and_empty():
    x, g = torch.randn(4, 64, device=DEV), torch.ones(64, device=DEV)
    y, m, r = ops.layernorm_train(x, g, g)
    for bad in (lambda: ops.layernorm_train(x.t(), g[:4], g[:4]), lambda: ops.layernorm_train(x, g[:32], g), lambda: ops.layernorm_train(x, g.bfloat16(), g),
                lambda: ops.layernorm_train(torch.zeros(2, 12296, device=DEV), torch.ones(12296, device=DEV), torch.ones(12296, device=DEV)),
                lambda: ops.layernorm_backward(x[:3], x, g, m, r), lambda: ops.layernorm_backward(x, x, g, m[:3], r),
                lambda: ops.layernorm_backward(x.t().contiguous().t(), x, g, m, r), lambda: ops.layernorm_backward(x[:, :1].expand(4, 64), x, g, m, r),
                lambda: ops.layernorm_backward(x, x, g, m, r, residual=x.bfloat16()), lambda: ops.layernorm_backward(x.cpu(), x, g, m, r)):
        with pytest.raises(_lib.SdamdError):
            bad()
    with pytest.raises(TypeError):
        ops.layernorm_train(x.half(), g, g)
    e = torch.empty(0, 64, device=DEV)
    ye, me, re_ = ops.layernorm_train(e, g, g)
    dx, dg, db = ops.layernorm_backward(e, e, g, me, re_)
    assert ye.shape == dx.shape == (0, 64) and not dg.any() and not db.any() and me.shape == (0,)


def test_layernorm_row_of_nan_stays_alone():
    x = rnd(1, (9, 640))
    x[4, 7] = float("nan")
    x[5] = 2.5                                       # no variance at all
    g = torch.ones(640, device=DEV)
    y, mean, rstd = ops.layernorm_train(x.to(DEV), g, 0 * g)
    assert y[4].isnan().all() and not y[[0, 1, 2, 3, 5, 6, 7, 8]].isnan().any()
    assert float(rstd[5]) == pytest.approx(1e-5 ** -0.5, rel=1e-6) and float(y[5].abs().max()) == 0.0
    dy = rnd(2, (9, 640)).to(DEV)
    dx, dg, db = ops.layernorm_backward(dy, x.to(DEV), g, mean, rstd)
    assert dx[4].isnan().all() and not dx[[0, 1, 2, 3, 5, 6, 7, 8]].isnan().any() and not db.isnan().any()


# ------------------------------------------------------------------ GeGLU
def geglu_ref(v, g):
    from scipy.special import ndtr
    return v * g * ndtr(g), g * ndtr(g), ndtr(g) + g * np.exp(-g * g / 2) / math.sqrt(2 * math.pi)


@pytest.mark.parametrize("rows,F", [(1, 1), (3, 7), (2, 64), (5, 100), (9, 128), (4, 129), (33, 320), (6, 1280), (3, 515)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("fmt", [E4M3, E5M2])
def test_geglu_train_and_backward(rows, F, dtype, fmt):
    h, dout = rnd(rows + F, (rows, 2 * F), dtype, 1.5), rnd(F, (rows, F), dtype, 0.1)
    out, kept = ops.geglu_train(h.to(DEV), fmt)
    H = np64(h)
    want, _, _ = geglu_ref(H[:, :F], H[:, F:])
    # erf is good to 1.5e-7 (7.5e-8 in Phi) and the exponential in it to a few roundings: 4e-7 in Phi and in phi(x) x
    half = UB if dtype == BF16 else 0
    close(out, want, 4e-7 * np.abs(H[:, :F] * H[:, F:]) + 4 * U * np.abs(want) + half * np.abs(want), "out")
    two = ops.quantize8(h.to(DEV), fmt)
    assert torch.equal(kept.q.view(torch.uint8), two.q.view(torch.uint8)) and torch.equal(kept.scale, two.scale)
    for given, vals in ((kept, np64(kept.dequantize(F32))), (h.to(DEV), H)):
        dh = ops.geglu_backward(dout.to(DEV), given)
        v, g, d = vals[:, :F], vals[:, F:], np64(dout)
        _, gelu, slope = geglu_ref(v, g)
        wv, wg = d * gelu, d * v * slope
        close(np64(dh)[:, :F], wv, 4e-7 * np.abs(d * g) + (4 * U + half) * np.abs(wv), "dvalue")
        close(np64(dh)[:, F:], wg, 8e-7 * np.abs(d * v) + (4 * U + half) * np.abs(wg), "dgate")
    other = BF16 if dtype == F32 else F32
    mixed = ops.geglu_backward(dout.to(DEV), kept, out_dtype=other)
    assert mixed.dtype == other
    if other == BF16:
        assert torch.equal(mixed, ops.geglu_backward(dout.to(DEV), kept).to(BF16))


@pytest.mark.parametrize("rows,F", [(1, 1), (3, 7), (2, 64), (5, 100), (9, 128), (4, 129), (33, 320), (6, 1280), (3, 515), (70, 384)])
@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("fmt", [E4M3, E5M2])
def test_geglu_train_into_blocks(rows, F, dtype, fmt):
    h = rnd(rows + F, (rows, 2 * F), dtype, 1.5)
    dense, kept = ops.geglu_train(h.to(DEV))
    out, kept2 = ops.geglu_train(h.to(DEV), out_dtype=fmt)
    assert out.shape == (rows, F) and out.dtype == fmt and out.block_rows == 1
    assert torch.equal(kept.q.view(torch.uint8), kept2.q.view(torch.uint8)) and torch.equal(kept.scale, kept2.scale)
    assert (out.q.view(torch.uint8)[:, F:] == 0).all()
    if dtype == F32:                                 # the same float32 products, quantised here or afterwards
        two = ops.quantize8(dense, fmt)
        assert torch.equal(out.q.view(torch.uint8), two.q.view(torch.uint8)) and torch.equal(out.scale, two.scale)
    H = np64(h)
    want, _, _ = geglu_ref(H[:, :F], H[:, F:])
    off = 4e-7 * np.abs(H[:, :F] * H[:, F:]) + 4 * U * np.abs(want)        # of the product itself, as above
    scale = np.repeat(2.0 ** scales_of(out), 128, 1)[:, :F]
    half, low, top = (2.0 ** -4, 2.0 ** -10, 448.0) if fmt == E4M3 else (2.0 ** -3, 2.0 ** -17, 57344.0)     # half a step: relative, and of the smallest numbers
    close(np64(out.dequantize(F32)), want, off + half * (np.abs(want) + off) + low * scale, "blocks")
    for b in range(-(-F // 128)):                    # the smallest scale that the product, as exact as it is, fits
        part, slack, s = np.abs(want[:, b * 128:b * 128 + 128]), off[:, b * 128:b * 128 + 128], scale[:, b * 128]
        assert ((part - slack).max(1) <= top * s).all() and ((part + slack).max(1) > top * s / 2).all()


@pytest.mark.parametrize("rows,F", [(1, 128), (5, 384), (300, 640), (3, 1), (7, 200), (0, 128)])
@pytest.mark.parametrize("out", [F32, BF16])
@pytest.mark.parametrize("fmt", [E4M3, E5M2])
def test_geglu_backward_with_blocks(rows, F, out, fmt):
    h, dout = rnd(rows + F, (rows, 2 * F), BF16, 1.5).to(DEV), rnd(F, (rows, F), BF16, 0.1).to(DEV)
    if rows > 2:
        h[1, 0], h[2, -1] = float("inf"), float("nan")
    kept = ops.quantize8(h)
    for given in (h, kept):
        want = ops.geglu_backward(dout, given, out_dtype=out)
        dh, d8 = ops.geglu_backward(dout, given, out_dtype=out, blocks=fmt)
        two = ops.quantize8(want, fmt)
        assert torch.equal(dh.nan_to_num(7.0), want.nan_to_num(7.0)) and d8.shape == (rows, 2 * F) and d8.dtype == fmt
        assert torch.equal(d8.q.view(torch.uint8), two.q.view(torch.uint8)) and torch.equal(d8.scale, two.scale)
    with pytest.raises(TypeError):
        ops.geglu_backward(dout, h, blocks=BF16)


def test_geglu_gradient_against_differences():
    rows, F, step = 3, 50, 1e-5
    h, dout = rnd(1, (rows, 2 * F)), rnd(2, (rows, F))
    dh = np64(ops.geglu_backward(dout.to(DEV), h.to(DEV)))
    H, D = np64(h), np64(dout)
    loss = lambda a: float((geglu_ref(a[:, :F], a[:, F:])[0] * D).sum())  # noqa: E731
    v = np.random.default_rng(1).standard_normal(H.shape)
    fd = (loss(H + step * v) - loss(H - step * v)) / (2 * step)
    assert abs((dh * v).sum() - fd) <= 1e-6 * np.abs(dh * v).sum() + 1e-7


def test_geglu_refusals_and_empty():
    h, d = torch.randn(4, 64, device=DEV), torch.randn(4, 32, device=DEV)
    for bad in (lambda: ops.geglu_train(h[:, :63]), lambda: ops.geglu_train(h[:, :62]), lambda: ops.geglu_backward(d[:3], h),
                lambda: ops.geglu_backward(d, h[:, ::2]), lambda: ops.geglu_backward(d.cpu(), h)):
        with pytest.raises(_lib.SdamdError):
            bad()
    with pytest.raises(TypeError):
        ops.geglu_backward(d.half(), h)
    for bad in (BF16, torch.float16, torch.int8):
        with pytest.raises(TypeError):
            ops.geglu_train(h, out_dtype=bad)
    assert ops.geglu_train(torch.empty(0, 64, device=DEV), out_dtype=E4M3)[0].shape == (0, 32)
    out, kept = ops.geglu_train(torch.empty(0, 64, device=DEV))
    assert out.shape == (0, 32) and ops.geglu_backward(torch.empty(0, 32, device=DEV), kept).shape == (0, 64)


# ------------------------------------------------------------------ together
def ffn_step(x, w1, b1, w2, b2, gamma, beta, dy, w1t, w2t):
    """Forward and backward of x + linear_2(geglu(linear_1(norm(x)))), everything kept for the backward pass in 8 bits."""
    n8, mean, rstd = ops.layernorm_train(x, gamma, beta, 1e-5, E4M3)
    h = ops.linear8(n8, w1, b1)
    g, h8 = ops.geglu_train(h)
    g8 = ops.quantize8(g)
    y = ops.linear8(g8, w2, b2, residual=x, out_dtype=F32)
    dyb = dy.to(BF16)
    dw2, db2 = ops.linear8_weight_grad(dyb, g8)
    dg = ops.linear8(dyb, w2t, fmt=E5M2)
    dh, dh8 = ops.geglu_backward(dg, h8, blocks=E5M2)
    dw1, db1 = ops.linear8_weight_grad(dh, n8)
    dn = ops.linear8(dh8, w1t)
    dx, dgamma, dbeta = ops.layernorm_backward(dn, x, gamma, mean, rstd, residual=dy)
    return y, dx, dw1, db1, dw2, db2, dgamma, dbeta


def ffn_inputs(rows, C, F, seed=0):
    x, dy = rnd(seed, (rows, C)), rnd(seed + 1, (rows, C), scale=0.1)
    w1, w2 = rnd(seed + 2, (2 * F, C), scale=C ** -0.5), rnd(seed + 3, (C, F), scale=F ** -0.5)
    b1, b2 = 0.1 * rnd(seed + 4, (2 * F,)), 0.1 * rnd(seed + 5, (C,))
    gamma, beta = 1 + 0.1 * rnd(seed + 6, (C,)), 0.1 * rnd(seed + 7, (C,))
    x, dy, w1, w2, b1, b2, gamma, beta = (t.to(DEV) for t in (x, dy, w1, w2, b1, b2, gamma, beta))
    return x, ops.quantize8_weight(w1), b1, ops.quantize8_weight(w2), b2, gamma, beta, dy, ops.quantize8_weight(w1.t()), ops.quantize8_weight(w2.t())


@pytest.mark.parametrize("rows,C,F", [(300, 320, 640), (77, 200, 260)])
def test_feed_forward_step(rows, C, F):
    """The operators as a training step runs them, against autograd in 64 bits on the unquantised problem.  Every 8-bit
    rounding is off by at most 2^-4 (e4m3) or 2^-3 (e5m2) of a value, uniformly spread: rms 2^-4 / sqrt(3) = 3.6 % or
    7.2 %; weights and activations enter each product once, so a result carries a few of them in quadrature."""
    inp = ffn_inputs(rows, C, F)
    got = ffn_step(*inp)
    x, w1, b1, w2, b2, gamma, beta, dy = inp[:8]
    d = torch.float64
    with torch.enable_grad():
        leaves = [t.cpu().to(d).requires_grad_() for t in (x, w1.dequantize(F32), b1, w2.dequantize(F32), b2, gamma, beta)]
        X, W1, B1, W2, B2, G, B = leaves
        n = torch.nn.functional.layer_norm(X, (C,), G, B, 1e-5)
        h = n @ W1.t() + B1
        y = X + (h[:, :F] * torch.nn.functional.gelu(h[:, F:])) @ W2.t() + B2
        y.backward(dy.cpu().to(d))
    want = (y.detach(), X.grad, W1.grad, B1.grad, W2.grad, B2.grad, G.grad, B.grad)
    for name, a, b in zip(("y", "dx", "dw1", "db1", "dw2", "db2", "dgamma", "dbeta"), got, want):
        rel = float((a.cpu().to(d) - b).norm() / b.norm())
        assert rel < 0.2, (name, rel)
    assert torch.allclose(got[5].cpu().to(d), dy.to(BF16).cpu().to(d).sum(0), rtol=0, atol=rows * U * float(dy.abs().sum(0).max()))


def test_feed_forward_step_on_another_stream_and_in_graphs():
    """The same bits on a side stream, in two captured graphs replayed in turn with eager work between, and from two
    streams at once: no scratch is shared."""
    a, b = ffn_inputs(130, 320, 384), ffn_inputs(260, 200, 136, 50)
    want_a, want_b = [t.clone() for t in ffn_step(*a)], [t.clone() for t in ffn_step(*b)]
    torch.cuda.synchronize()
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    for _ in range(3):
        with torch.cuda.stream(s1):
            ra = ffn_step(*a)
        with torch.cuda.stream(s2):
            rb = ffn_step(*b)
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip(ra, want_a)) and all(torch.equal(x, y) for x, y in zip(rb, want_b))
    graphs = []
    for inp in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            res = ffn_step(*inp)
        graphs.append((g, res))
    for _ in range(3):
        for (g, res), want in zip(graphs, (want_a, want_b)):
            for t in res:
                t.zero_()
            g.replay()
            eager = ffn_step(*a)
            torch.cuda.synchronize()
            assert all(torch.equal(x, y) for x, y in zip(res, want)) and all(torch.equal(x, y) for x, y in zip(eager, want_a))


def test_results_past_the_cache_are_the_same():
    """Results of 128 MB or more are written another way than small ones: the same bits as in parts."""
    w = ops.quantize8_weight(rnd(4, (4100, 130)).to(DEV))
    for out, M in ((BF16, 16500), (F32, 8250)):
        x = ops.quantize8(rnd(3, (M, 130)).to(DEV))
        whole = ops.linear8(x, w, out_dtype=out)
        assert whole.numel() * whole.element_size() >= 1 << 27
        for at in range(0, M, M // 3):
            part = ops.Blocks8(x.q[at:at + M // 3], x.scale[at:at + M // 3], (M // 3, 130))
            assert torch.equal(whole[at:at + M // 3], ops.linear8(part, w, out_dtype=out))
    for F, rows in ((1280, 52500), (129, 260400)):
        h, d = rnd(1, (rows, 2 * F)).to(DEV), rnd(2, (rows, F)).to(DEV)
        out, kept = ops.geglu_train(h)
        dh = ops.geglu_backward(d, kept)
        for at in (0, rows - 500):
            o, k = ops.geglu_train(h[at:at + 500])
            assert torch.equal(out[at:at + 500], o) and torch.equal(kept.q[at:at + 500].view(torch.uint8), k.q.view(torch.uint8))
            assert torch.equal(dh[at:at + 500], ops.geglu_backward(d[at:at + 500], k))


def test_writes_stay_inside():
    """Outputs cut from one buffer with guard values on both sides: nothing outside them is written."""
    def guarded(n, dtype):
        buf = torch.full((n + 512,), 7.0, dtype=dtype, device=DEV)
        return buf, buf[256:256 + n]
    L = _lib.lib()
    st = lambda: torch.cuda.current_stream().cuda_stream  # noqa: E731
    for M, N, K in ((5, 19, 130), (70, 45, 200), (300, 1300, 129), (2500, 2300, 140)):
        x8, w8 = ops.quantize8(rnd(1, (M, K)).to(DEV)), ops.quantize8_weight(rnd(2, (N, K)).to(DEV))
        for dt, code in ((BF16, 1), (F32, 0)):
            buf, out = guarded(M * N, dt)
            _lib.check(L.sdamd_linear8(x8.q.data_ptr(), x8.scale.data_ptr(), w8.q.data_ptr(), w8.scale.data_ptr(), out.data_ptr(), 0, 0,
                                       M, N, K, 0, 2, 2, code, st()))
            assert torch.equal(out.view(M, N), ops.linear8(x8, w8, out_dtype=dt)) and (buf[:256] == 7).all() and (buf[-256:] == 7).all()
    for T, N, K in ((9, 19, 130), (700, 264, 257)):
        x8, dy = ops.quantize8(rnd(1, (T, K)).to(DEV)), rnd(2, (T, N), BF16).to(DEV)
        bw, dw = guarded(N * K, F32)
        bb, db = guarded(N, F32)
        need = L.sdamd_linear8_weight_grad_ws_bytes(T, N, K)
        ws = torch.empty(max(need, 1), dtype=torch.uint8, device=DEV)
        _lib.check(L.sdamd_linear8_weight_grad(dy.data_ptr(), x8.q.data_ptr(), x8.scale.data_ptr(), dw.data_ptr(), db.data_ptr(), ws.data_ptr(), need,
                                               T, N, K, 2, st()))
        w, b = ops.linear8_weight_grad(dy, x8)
        assert torch.equal(dw.view(N, K), w) and torch.equal(db, b)
        assert all((t[:256] == 7).all() and (t[-256:] == 7).all() for t in (bw, bb))
    for rows, C in ((3, 77), (40, 320), (5, 5000)):
        x, g = rnd(1, (rows, C)).to(DEV), torch.ones(C, device=DEV)
        for dt, code in ((BF16, 1), (F32, 0)):
            by, y = guarded(rows * C, dt)
            bm, mean = guarded(rows, F32)
            br, rstd = guarded(rows, F32)
            _lib.check(L.sdamd_layernorm_train(x.data_ptr(), y.data_ptr(), 0, g.data_ptr(), g.data_ptr(), mean.data_ptr(), rstd.data_ptr(), rows, C,
                                               1e-5, 0, code, st()))
            assert all((t[:256] == 7).all() and (t[-256:] == 7).all() for t in (by, bm, br))


# ------------------------------------------------------------------ Linear's activations over their whole range
def activation_sweep(dtype):
    """Pre-activations from one end of the type to the other, dense around -52.1 and -88.7, where the exponential in x / (1 +
    exp(-c x)) leaves float32's range for c = 1.702 and 1, and what f32 arithmetic gives there in 64 bits."""
    v = np.concatenate([np.arange(-1000, 1000, 0.37), np.arange(-130, -40, 0.01), np.arange(-1, 1, 1e-3),
                        np.linspace(-1e4, 1e4, 401), np.array([0.0, -0.0, 1e-30, -1e-30, 1e30, -1e30, 3e38, -3e38, np.inf, -np.inf, np.nan])])
    return torch.from_numpy(v).to(dtype)


def activation_ref(v, act):
    """(value, bound) of x / (1 + exp(-c x)) for an exact x: the exponential 1 ulp, the digits that its argument lost put back in two
    roundings, 1 + e half a step, the reciprocal 1 ulp, the product half a step: (2 + 2) + 1 + 2 + 1 = 8 U.  c = 1.702 is a
    rounded constant and c x a rounded product, which the exponential carries on as 2 U |c x|.  A reciprocal below the smallest
    normal number 2^-126 may come out as zero (only where |x| < 200)."""
    c = 1.0 if act == ops.ACT_SILU else 1.702
    with np.errstate(over="ignore", invalid="ignore"):
        want = v / (1 + np.exp(-c * v))
        tol = (8 * U + (0 if act == ops.ACT_SILU else 2 * U * np.minimum(np.abs(c * v), 200))) * np.abs(want) + np.minimum(np.abs(v), 200) * 2.0 ** -126
    return want, tol


# (M, N): the rows kernel with 16, 32 and 64 rows a workgroup, the 128 x 128 tile whole and ragged, the 256 x 256 tile (bf16)
# whole and ragged
@pytest.mark.parametrize("M,N", [(16, 200), (30, 333), (200, 333), (2048, 1024), (1500, 2050), (4096, 4096), (4100, 3501)])
@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("act", [ops.ACT_SILU, ops.ACT_QUICK_GELU])
def test_linear8_activation_over_its_range(M, N, out, act):
    """Rows of zeros: the residual, or the bias, is the pre-activation."""
    w, x = ops.quantize8_weight(rnd(1, (N, 40)).to(DEV)), torch.zeros(M, 40, device=DEV)
    x8 = ops.quantize8(x)
    v = activation_sweep(out)
    res = v.repeat(-(-M * N // v.numel()))[:M * N].view(M, N).to(DEV)
    bias = activation_sweep(F32).flip(0)
    bias = bias.repeat(-(-N // bias.numel()))[torch.randperm(max(N, bias.numel()), generator=gen(N))[:N]].to(DEV)
    for pre, got in ((res, ops.linear8(x, w, None, res, act, out)), (res, ops.linear8(x8, w, None, res, act, out)),
                     (bias.expand(M, N), ops.linear8(x8, w, bias, None, act, out))):
        pre, got = np64(pre), np64(got)
        want, tol = activation_ref(pre, act)
        if out == BF16:
            tol = tol + UB * np.abs(want)
        fin = np.isfinite(pre)
        close(got[fin], want[fin], tol[fin], f"act {act}")
        assert np.array_equal(got[~fin], want[~fin], equal_nan=True)         # inf -> inf, NaN -> NaN, -inf 0 -> NaN


# ------------------------------------------------------------------ the sums inside the 8-bit matrix instruction
def spread8(seed, shape, low, high):
    """Magnitudes over high - low octaves: products of very different size beside one another."""
    g = gen(seed)
    return torch.randn(shape, generator=g) * torch.exp2(torch.randint(low, high, shape, generator=g).float())


def instruction_sum(x, w):
    """(what the 8-bit instruction makes of x @ w.T: products of 8 consecutive k cut toward zero at 2^-13 of the largest power of two
    among them, the exact sum, the sum of magnitudes) in 64 bits."""
    prod = (x[:, None, :] * w[None]).reshape(len(x), len(w), -1, 8)
    power = lambda v: np.where(v == 0, -2000, np.frexp(v)[1] - 1)  # noqa: E731
    top = (power(x)[:, None, :] + power(w)[None]).reshape(prod.shape).max(-1, keepdims=True)
    step = np.ldexp(1.0, np.maximum(top - 13, -1000))
    return (np.trunc(prod / step) * step).sum((-1, -2)), prod.sum((-1, -2)), np.abs(prod).sum((-1, -2))


# the rows kernel with 16, 32 and 64 rows a workgroup, the 128 x 128 and the 256 x 256 tile (bf16; float32 results have no such tile)
@pytest.mark.parametrize("M,K,N", [(16, 128, 64), (30, 640, 40), (64, 384, 96), (200, 256, 333), (1024, 256, 1024), (4096, 128, 4096)])
@pytest.mark.parametrize("fmt", [E4M3, E5M2])
def test_linear8_sums_are_what_is_documented(M, K, N, fmt):
    x8, w8 = ops.quantize8(spread8(1, (M, K), -9, 6).to(DEV), fmt), ops.quantize8_weight(spread8(2, (N, K), -6, 6).to(DEV))
    rows, cols = np.unique(np.r_[0:20, max(M - 20, 0):M].clip(max=M - 1)), np.r_[0:20, N - 20:N]
    cut, exact, mag = instruction_sum(np64(x8.dequantize(F32))[rows], np64(w8.dequantize(F32))[cols])
    # 16 groups a block and the blocks are added with 23 bits below the largest
    adds = 17 * (K // 128) * 2.0 ** -23 * mag
    close(np64(ops.linear8(x8, w8, out_dtype=BF16))[rows][:, cols], cut, UB * np.abs(cut) + adds, "bf16")
    close(np64(ops.linear8(x8, w8, out_dtype=F32))[rows][:, cols], exact, (K + 4) * U * mag, "f32")


@pytest.mark.parametrize("M,N", [(3, 16), (1024, 1024), (4096, 4096)])
def test_linear8_products_that_cancel(M, N):
    """256 * 256 - 256 * 256 + 2^(16 - d) in one group of 8, and the small one in a group of its own."""
    for at, kept in ((2, 13), (8, 23)):
        for d in (4, 12, 13, 14, 20):
            x, w = torch.zeros(M, 128), torch.zeros(N, 128)
            x[:, :2], w[:, 0], w[:, 1] = 256.0, 256.0, -256.0
            x[:, at], w[:, at] = 2.0 ** (8 - d // 2), 2.0 ** (8 - (d - d // 2))
            x8, w8 = ops.quantize8(x.to(DEV)), ops.quantize8_weight(w.to(DEV))
            assert (ops.linear8(x8, w8, out_dtype=F32) == 2.0 ** (16 - d)).all()
            got = ops.linear8(x8, w8, out_dtype=BF16)
            assert (got <= 2.0 ** (16 - d)).all() and (got >= (2.0 ** (16 - d) if d <= kept else 0.0)).all(), (at, d)


# one width for each form of the kernel (lanes a row, vectors a lane), all but one of them ragged; rows that give a workgroup of the
# form's RP rows two or three turns, the last of them short
LNB_FORMS = [(65, 64, 599), (190, 64, 299), (333, 32, 599), (500, 16, 599), (700, 16, 299), (1001, 8, 299), (1500, 8, 299), (2047, 8, 599),
             (4095, 2, 299), (8191, 1, 299), (12288, 1, 300)]


@pytest.mark.parametrize("C,RP,turns", LNB_FORMS)
@pytest.mark.parametrize("xt,dt,skip", [(F32, F32, True), (BF16, BF16, False), (E4M3, BF16, True), (E5M2, F32, False)])
def test_layernorm_backward_joins_many_rows(C, RP, turns, xt, dt, skip):
    """Weight gradients through partial sums: every form of the kernel, workgroups with several turns, x of every type."""
    rows = RP * turns - RP // 2
    assert _lib.lib().sdamd_layernorm_backward_ws_bytes(rows, C) == -(-turns // -(-turns // 256)) * 8 * C       # (so many workgroups leave partial sums)
    x = rnd(C, (rows, C)) + 0.5
    dy, gamma = rnd(C + 1, (rows, C), dt, 0.1), 1 + 0.2 * rnd(3, (C,))
    if xt in (E4M3, E5M2):
        given = ops.quantize8(x.to(DEV), xt)
        vals, ot = given.dequantize(F32), dt
    else:
        given = vals = x.to(xt).to(DEV)
        ot = xt
    res = rnd(9, (rows, C), ot) if skip else None
    _, mean, rstd = ops.layernorm_train(vals, gamma.to(DEV), torch.zeros(C, device=DEV))
    call = lambda: ops.layernorm_backward(dy.to(DEV), given, gamma.to(DEV), mean, rstd, None if res is None else res.to(DEV))  # noqa: E731
    dx, dg, db = call()
    w_dx, w_dg, w_db, tol, e_g, mag_g = backward_ref(np64(dy), np64(vals), np64(gamma), None if res is None else np64(res), 1e-5)
    close(dx, w_dx, tol + (UB * np.abs(w_dx) if ot == BF16 else 0), "dx")
    # a column's sum: at most 3 rows after one another, 3 shuffles, 1 + 3 over the waves, 16 partial rows and 16 lanes of them
    close(dg, w_dg, e_g + 48 * U * mag_g, "dgamma")
    close(db, w_db, 48 * U * np.abs(np64(dy)).sum(0), "dbeta")
    assert all(torch.equal(a, b) for a, b in zip(call(), (dx, dg, db)))          # the same bits every run


@pytest.mark.parametrize("out", [BF16, F32])
@pytest.mark.parametrize("M", [5, 64, 1100])
def test_linear8_out_beside_its_operands(M, out):
    """x, bias, residual and out from one buffer: next to one another they are taken, one element into one another refused; out may
    be the residual."""
    K, N = 256, 320
    es = torch.empty(0, dtype=out).element_size()
    w = ops.quantize8_weight(rnd(1, (N, K)).to(DEV))
    x, res, bias = rnd(2, (M, K), out).to(DEV), rnd(3, (M, N), out).to(DEV), rnd(4, (N,)).to(DEV)
    want = ops.linear8(x, w, bias, res, out_dtype=out)
    buf = torch.empty((M * K + 2 * M * N) * es + N * 4, dtype=torch.uint8, device=DEV)
    cut = lambda at, n, dtype, shape: buf[at:at + n * torch.empty(0, dtype=dtype).element_size()].view(dtype).view(shape)  # noqa: E731
    def fill():
        xs, bs = cut(0, M * K, out, (M, K)), cut((M * K + M * N) * es, N, F32, (N,))
        rs = cut((M * K + M * N) * es + N * 4, M * N, out, (M, N))
        return xs.copy_(x), bs.copy_(bias), rs.copy_(res)
    xs, bs, rs = fill()
    o = cut(M * K * es, M * N, out, (M, N))
    assert torch.equal(ops.linear8(xs, w, bs, rs, out_dtype=out, out=o), want)
    assert torch.equal(ops.linear8(xs, w, bs, rs, out_dtype=out, out=rs), want)
    xs, bs, rs = fill()
    keep = buf.clone()
    for at in (-es, es):                                 # into x's end, into the bias
        bad = cut(M * K * es + at, M * N, out, (M, N))
        with pytest.raises(_lib.SdamdError, match="overlaps"):
            ops.linear8(xs, w, bs, rs, out_dtype=out, out=bad)
    bad = cut((M * K + M * N) * es + N * 4 - es, M * N, out, (M, N))     # one element before the residual
    with pytest.raises(_lib.SdamdError, match="overlaps"):
        ops.linear8(xs, w, None, rs, out_dtype=out, out=bad)
    x8 = ops.quantize8(xs)
    row = ops.Blocks8(x8.q[:1], x8.scale[:1], (1, K))
    with pytest.raises(_lib.SdamdError, match="overlaps"):
        ops.linear8(row, w, out=x8.q.view(-1)[128:128 + 2 * N].view(BF16).view(1, N))
    assert torch.equal(buf, keep)                        # nothing was written


# ------------------------------------------------------------------ offsets that pass 32 bits
BIG = 180000, 12288                                      # 2.2e9 elements


def big(seed, shape, dtype=BF16):
    return torch.randn(shape, generator=torch.Generator(device=DEV).manual_seed(seed), device=DEV, dtype=dtype)


def same_rows(whole, rows, part):
    """The last rows of a long result and the result of those rows alone."""
    if isinstance(whole, ops.Blocks8):
        n = part.q.shape[0]
        return torch.equal(whole.q[-n:].view(torch.uint8), part.q.view(torch.uint8)) and torch.equal(whole.scale[-n:], part.scale)
    return torch.equal(whole[-rows:], part)


def test_long_rows_quantised_and_normalised():
    R, C, n = *BIG, 9
    x = big(1, (R, C))
    x8 = ops.quantize8(x)
    assert same_rows(x8, n, ops.quantize8(x[-n:])) and same_rows(x8.dequantize(), n, ops.quantize8(x[-n:]).dequantize())
    g, b = 1 + 0.1 * big(2, (C,), F32), big(3, (C,), F32)
    y, mean, rstd = ops.layernorm_train(x, g, b)
    ys, ms, rs = ops.layernorm_train(x[-n:], g, b)
    assert same_rows(y, n, ys) and same_rows(mean, n, ms) and same_rows(rstd, n, rs)
    assert same_rows(ops.layernorm_train(x, g, b, out_dtype=E4M3)[0], n, ops.layernorm_train(x[-n:], g, b, out_dtype=E4M3)[0])
    for given, part in ((x, x[-n:]), (x8, ops.quantize8(x[-n:]))):
        dx = ops.layernorm_backward(y, given, g, mean, rstd, residual=x)[0]
        assert same_rows(dx, n, ops.layernorm_backward(ys, part, g, ms, rs, residual=x[-n:])[0])


@pytest.mark.parametrize("F", [6144, 6143])
def test_long_rows_geglu(F):
    n = 9
    h = big(1, (BIG[0], 2 * F))
    out, kept = ops.geglu_train(h)
    po, pk = ops.geglu_train(h[-n:])
    assert same_rows(out, n, po) and same_rows(kept, n, pk)
    assert same_rows(ops.geglu_train(h, out_dtype=E4M3)[0], n, ops.geglu_train(h[-n:], out_dtype=E4M3)[0])
    dh, d8 = ops.geglu_backward(out, kept, blocks=E5M2)
    pd, p8 = ops.geglu_backward(po, pk, blocks=E5M2)
    assert same_rows(dh, n, pd) and same_rows(d8, n, p8) and same_rows(ops.geglu_backward(out, h), n, ops.geglu_backward(po, h[-n:]))


@pytest.mark.parametrize("out", [BF16, F32])
def test_long_rows_linear(out):
    """Past 32 bits in the result and the residual, then in the rows; enough rows alone for the same kernel."""
    R, C, n = *BIG, 20000
    for K, N in ((100, C), (C, 16)):
        x8 = ops.quantize8(big(1, (R, K)))
        part = ops.Blocks8(x8.q[-n:], x8.scale[-n:], (n, K))
        w, res = ops.quantize8_weight(big(2, (N, K))), big(3, (R, N), out)
        whole = ops.linear8(x8, w, residual=res, out_dtype=out)
        assert same_rows(whole, n, ops.linear8(part, w, residual=res[-n:], out_dtype=out))
        del x8, res, whole


@pytest.mark.parametrize("N,K", [(BIG[1], 16), (16, BIG[1]), (BIG[1] - 3, 16)])
def test_long_weight_grad(N, K):
    """Whole numbers, so that sums are exact; only the last rows of dy are not zero."""
    T, n = BIG[0], 100
    dy, x = torch.zeros((T, N), dtype=BF16, device=DEV), torch.zeros((T, K), dtype=BF16, device=DEV)
    dy[-n:], x[-n:] = big(1, (n, N)).round(), big(2, (n, K)).round()
    x[:1000] = 3
    dw, db = ops.linear8_weight_grad(dy, ops.quantize8(x))
    w, b = ops.linear8_weight_grad(dy[-n:].contiguous(), ops.quantize8(x[-n:]))
    assert torch.equal(dw, w) and torch.equal(db, b) and bool(dw.any())
