"""CPU-only checks of the 8-bit and training operators: arguments are refused before anything is launched, at the C
boundary and in Python, and the host-side plans hold."""
import subprocess
import sys

import pytest
import torch

import sd_amd  # noqa: F401
from sd_amd import _lib, ops
from conftest import ROOT

L = _lib.lib()
P = 4096            # an address that is never read: every call below is refused on the host


def refused(rc, text):
    assert rc != 0 and text in L.sdamd_last_error().decode(), (rc, L.sdamd_last_error())


def test_c_boundary_refuses_bad_arguments():
    refused(L.sdamd_quant8(P, P, P, 0, 5, 5, 0, 2, 0), "bad shape")
    refused(L.sdamd_quant8(P, P, P, 4, 5, 5, 7, 2, 0), "unsupported dtypes")
    refused(L.sdamd_quant8(P, P, P, 4, 5, 5, 0, 1, 0), "unsupported dtypes")
    refused(L.sdamd_quant8(P, P, P, 1 << 40, 1280, 1280, 0, 2, 0), "too large")
    refused(L.sdamd_quant8_weight(P, P, P, 0, 5, 5, 1, 0, 0), "bad shape")
    refused(L.sdamd_quant8_weight(P, P, P, 5, 5, -1, 1, 0, 0), "bad shape")
    refused(L.sdamd_dequant8(P, P, P, 4, 5, 64, 2, 0, 0), "block_rows")
    refused(L.sdamd_dequant8(P, P, P, 4, 5, 1, 0, 0, 0), "unsupported dtypes")
    refused(L.sdamd_linear8(P, P, P, P, P, 0, 0, 0, 4, 4, 0, 2, 2, 1, 0), "bad shape")
    refused(L.sdamd_linear8(P, P, P, P, P, 0, 0, 4, 4, 4, 0, 3, 2, 1, 0), "unsupported dtypes")       # blocks of another type than fmt
    refused(L.sdamd_linear8(P, P, P, P, P, 0, 0, 4, 4, 4, 0, 2, 2, 2, 0), "unsupported dtypes")
    refused(L.sdamd_linear8(P, P, P, P, P, 0, 0, 4, 4, 4, 3, 2, 2, 1, 0), "activation")
    refused(L.sdamd_linear8(P, 0, P, P, P, 0, 0, 4, 4, 4, 0, 2, 2, 1, 0), "without their scales")
    refused(L.sdamd_linear8(P, 0, P, P, P, 0, 0, 9000, 4096, 4096, 0, 1, 2, 1, 0), "quantised first")
    assert L.sdamd_linear8_quantises(1, 1280, 320, 1) == 1 and L.sdamd_linear8_quantises(9000, 4096, 4096, 1) == 0 and L.sdamd_linear8_quantises(0, 1, 1, 0) == 0
    refused(L.sdamd_linear8(P, P, P, P, P, 0, 0, 4, 4, (1 << 24) + 1, 0, 2, 2, 1, 0), "bad shape")
    refused(L.sdamd_linear8(P + 8, P, P, P, P, 0, 0, 4, 4, 4, 0, 2, 2, 1, 0), "aligned")
    refused(L.sdamd_linear8(P, P + 2, P, P, P, 0, 0, 4, 4, 4, 0, 2, 2, 1, 0), "aligned")
    refused(L.sdamd_linear8_weight_grad(P, P, P, P, P, 0, 0, 4, (1 << 24) + 1, 4, 2, 0), "bad shape")
    refused(L.sdamd_linear8_weight_grad(P, P + 4, P, P, P, 0, 0, 4, 4, 4, 2, 0), "aligned")
    refused(L.sdamd_layernorm_train(P, P, 0, P, P, P, P, 1 << 24, 768, 1e-5, 0, 0, 0), "too many rows")
    refused(L.sdamd_layernorm_backward(P, P, 0, P, P, P, 0, P, P, P, P, 1 << 30, 1 << 29, 8, 0, 0, 0, 0), "too many rows")
    refused(L.sdamd_geglu_train(P, P, 0, P, P, 1 << 40, 64, 0, 0, 2, 0), "too large")
    refused(L.sdamd_geglu_backward(P, P, 0, P, 0, 0, 1 << 40, 64, 0, 0, 0, 0, 0), "too large")
    refused(L.sdamd_linear8_weight_grad(P, P, P, P, P, 0, 0, 0, 4, 4, 2, 0), "bad shape")
    refused(L.sdamd_linear8_weight_grad(P, P, P, P, P, 0, 0, 4, 4, 4, 1, 0), "unsupported dtype")
    need = L.sdamd_linear8_weight_grad_ws_bytes(65536, 320, 320)
    assert need > 0
    refused(L.sdamd_linear8_weight_grad(P, P, P, P, P, P, need - 1, 65536, 320, 320, 2, 0), "workspace")
    refused(L.sdamd_layernorm_train(P, P, 0, P, P, P, P, 4, 12289, 1e-5, 0, 0, 0), "unsupported shape")
    refused(L.sdamd_layernorm_train(P, P, 0, P, P, P, P, 0, 64, 1e-5, 0, 0, 0), "unsupported shape")
    refused(L.sdamd_layernorm_train(P, P, 0, P, P, P, P, 4, 64, 1e-5, 0, 2, 0), "without room")
    refused(L.sdamd_layernorm_train(P, P, 0, P, P, P, P, 4, 64, 1e-5, 2, 0, 0), "unsupported dtypes")
    need = L.sdamd_layernorm_backward_ws_bytes(4, 64)
    many = L.sdamd_layernorm_backward_ws_bytes(4096, 64)
    refused(L.sdamd_layernorm_backward(P, P, 0, P, P, P, 0, P, P, P, P, many - 1, 4096, 64, 0, 0, 0, 0), "workspace")
    refused(L.sdamd_layernorm_backward(P, P, 0, P, P, P, 0, P, P, P, P, need, 4, 64, 0, 2, 0, 0), "without its scales")
    refused(L.sdamd_layernorm_backward(P, P, 0, P, P, P, 0, P, P, P, P, need, 4, 64, 2, 0, 0, 0), "unsupported dtypes")
    refused(L.sdamd_geglu_train(P, P, 0, P, P, 0, 64, 0, 0, 2, 0), "bad shape")
    refused(L.sdamd_geglu_train(P, P, 0, P, P, 4, 64, 2, 2, 2, 0), "unsupported dtypes")
    refused(L.sdamd_geglu_train(P, P, 0, P, P, 4, 64, 1, 0, 2, 0), "unsupported dtypes")
    refused(L.sdamd_geglu_train(P, P, 0, P, P, 4, 64, 0, 2, 2, 0), "without room")
    refused(L.sdamd_geglu_backward(P, P, 0, P, 0, 0, 4, 64, 0, 2, 0, 0, 0), "without its scales")
    refused(L.sdamd_geglu_backward(P, P, 0, P, 0, 0, 4, 64, 2, 0, 0, 0, 0), "unsupported dtypes")
    for args in ((P, 0, 4, 128, 0, 0, 1, 2), (P, P, 4, 128, 0, 0, 0, 2), (P, P, 4, 64, 0, 0, 1, 2), (P, P, 4, 128, 0, 0, 1, 1)):
        refused(L.sdamd_geglu_backward(P, P, 0, P, *args, 0), "blocks of dh")


def test_c_boundary_keeps_launches_below_2_to_32_threads():
    refused(L.sdamd_quant8(P, P, P, (1 << 29) - 31, 8, 8, 0, 2, 0), "too large")
    refused(L.sdamd_dequant8(P, P, P, (1 << 28) - 15, 8, 1, 2, 0, 0), "too large")
    refused(L.sdamd_geglu_train(P, P, 0, P, P, 1 << 30, 4, 0, 0, 2, 0), "too large")
    refused(L.sdamd_geglu_train(P, P, P, P, P, 1 << 30, 128, 0, 3, 2, 0), "too large")
    refused(L.sdamd_layernorm_train(P, P, 0, P, P, P, P, (1 << 27) - 31, 512, 1e-5, 0, 0, 0), "too many rows")


def test_python_refuses_the_cpu_and_bad_blocks():
    x = torch.zeros(4, 200)
    for call in (lambda: ops.quantize8(x), lambda: ops.quantize8_weight(x), lambda: ops.layernorm_train(x, x[0], x[0]),
                 lambda: ops.layernorm_backward(x, x, x[0], x[:, 0], x[:, 0]), lambda: ops.geglu_train(x), lambda: ops.geglu_backward(x[:, :100], x)):
        with pytest.raises(_lib.SdamdError, match="HIP device"):
            call()
    q, s = torch.zeros(4, 256, dtype=torch.float8_e4m3fn), torch.full((4, 4), 127, dtype=torch.uint8)
    b = ops.Blocks8(q, s, (2, 2, 200))
    assert b.nbytes == 4 * 256 + 16 and b.dtype == torch.float8_e4m3fn
    for call in (lambda: b.dequantize(), lambda: ops.geglu_backward(torch.zeros(2, 2, 100), b)):
        with pytest.raises(_lib.SdamdError, match="HIP device"):
            call()
    bad = [(q, s, (4, 257), 1), (q, s, (5, 200), 1), (q[:, :128], s, (4, 128), 1), (q, s[:, :2], (4, 200), 1), (q, s.int(), (4, 200), 1),
           (q, s, (4, 200), 64), (q, s, (4, 200), 128), (q.view(torch.float8_e5m2), s[:1], (4, 200), 128), (q, s, (4, 0), 1),
           (torch.zeros(4 * 256 + 16, dtype=torch.uint8)[1:1025].view(torch.float8_e4m3fn).view(4, 256), s, (4, 200), 1)]
    for args in bad:
        with pytest.raises(_lib.SdamdError, match="Blocks8"):
            ops.Blocks8(*args)
    with pytest.raises(TypeError):
        ops.Blocks8(q.view(torch.int8), s, (4, 200))


def test_sizes_are_not_cut_at_the_boundary():
    """ctypes would pass 2^32 + 5 as 5."""
    ops._fits("x", 1, 0x7fffffff)
    with pytest.raises(_lib.SdamdError, match="too large"):
        ops._fits("x", 5, (1 << 32) + 5)


def test_workspaces_cover_their_plans():
    """Few tiles and many tokens are split; wide gradients and short ones are not."""
    ws = L.sdamd_linear8_weight_grad_ws_bytes
    assert ws(77, 320, 320) == 0 and ws(0, 4, 4) == 0
    for t, n, k in ((65536, 320, 320), (16384, 5120, 640), (4099, 333, 215)):
        per = (n * k + n) * 4
        assert ws(t, n, k) % per == 0 and ws(t, n, k) // per <= 512
    for rows, c in ((1, 1), (77, 768), (1 << 30, 320), (4099, 1001), (50000, 12288)):  # a row of partial sums per workgroup
        need = L.sdamd_layernorm_backward_ws_bytes(rows, c)
        assert need % (8 * c) == 0 and need <= min(rows, 512) * 8 * c and (need > 0) == (rows > 1000)
    assert L.sdamd_layernorm_backward_ws_bytes(4, 12289) == 0


def test_import_without_torch_s_private_names():
    """A torch without GPU support lacks the two shortcuts: the module is imported all the same, and the public calls take their
    place."""
    code = """
import torch
for name in ("_cuda_getDevice", "_cuda_getCurrentRawStream"):
    if hasattr(torch._C, name):
        delattr(torch._C, name)
import sd_amd
from sd_amd import _lib, diffusion, ops, pipeline
assert ops._current_device is torch.cuda.current_device
class Stream:
    cuda_stream = 1234
torch.cuda.current_stream = lambda i: Stream if i == 5 else None
assert ops._raw_stream(5) == 1234
try:
    ops.quantize8(torch.zeros(4, 200))
except _lib.SdamdError as e:
    assert "HIP device" in str(e)
else:
    raise AssertionError
"""
    subprocess.run([sys.executable, "-c", code], check=True, cwd=ROOT)


def test_linear8_out_overlaps_no_operand():
    """M = 70, N = 40, K = 200 (blocks of 256 bytes, 4 scale bytes), far apart but for the one that is named."""
    M, N, K = 70, 40, 200
    base = {"x": 1 << 32, "x_scale": 2 << 32, "w": 3 << 32, "w_scale": 4 << 32, "bias": 6 << 32, "residual": 7 << 32}
    out = 5 << 32
    for code, es in ((0, 4), (1, 2)):
        end = M * N * es
        size = {"x": M * 256, "x_scale": M * 4, "w": N * 256, "w_scale": 4, "bias": N * 4, "residual": end}
        for name, n in size.items():
            step = 16 if name in ("x", "w") else 4
            for at in (out + end - step, out - n + step) + ((out,) if name != "residual" else (out + step, out - step)):
                a = dict(base, **{name: at})
                refused(L.sdamd_linear8(a["x"], a["x_scale"], a["w"], a["w_scale"], out, a["bias"], a["residual"], M, N, K, 0, 2, 2, code, 0), "overlaps")
    for x_dtype, n in ((0, 4), (1, 2)):                  # rows that the kernel quantises itself
        refused(L.sdamd_linear8(out - 40 * K * n + n, 0, base["w"], base["w_scale"], out, 0, 0, 40, N, K, 0, x_dtype, 2, 1, 0), "overlaps")
    t = torch.zeros(100)
    assert ops._overlap(t[:50], t[49:]) and ops._overlap(t[10:20], t) and not ops._overlap(t[:50], t[50:]) and not ops._overlap(t[50:], t[:50])
