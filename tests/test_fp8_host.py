"""The 8-bit tensors, the linear layers on them and LayerNorm's training passes refuse bad calls on the host, before any
launch (CPU: the addresses are never dereferenced), and report the sizes their layout has."""
from __future__ import annotations

import ctypes

import pytest

torch = pytest.importorskip("torch")

OK, ODD8, ODD2, ODD1 = (ctypes.c_void_p((1 << 20) + d) for d in (0, 8, 2, 1))
BIG = 1 << 40


def _call(fvsr, name, good, **change):
    args = dict(good)
    args.update(change)
    status = getattr(fvsr.lib(), name)(*args.values())
    return status, fvsr.lib().fvsr_last_error()


QUANT = dict(rows=5, cols=9, x=OK, dtype=1, square=0, q=OK, scale=OK, qt=OK, scale_t=OK, stream=None)
DEQUANT = dict(rows=5, cols=9, q=OK, scale=OK, out=OK, dtype=1, stream=None)
CODES = dict(rows=5, cols=9, scale=OK, out=OK, stream=None)
LINEAR = dict(m=5, n=6, k=7, x=OK, x_scale=OK, w=OK, w_scale=OK, bias=OK, epilogue=2, gate=OK, resid=OK, out=OK,
              out_dtype=1, workspace=OK, workspace_bytes=BIG, stream=None)
NORM = dict(m=5, c=6, x=OK, dtype=1, weight=OK, bias=OK, shift=OK, scale=OK, eps=1e-6, out=OK, mean=OK, rstd=OK,
            stream=None)
BACK = dict(m=5, c=6, dy=OK, dtype=1, x=OK, x_scale=OK, mean=OK, rstd=OK, weight=OK, bias=OK, scale=OK, dx=OK,
            dweight=OK, dbias=OK, dscale=OK, dshift=OK, workspace=OK, workspace_bytes=BIG, stream=None)

REFUSED = [
    ("fvsr_quantize_fp8", QUANT, dict(rows=-1), 1, b"rows"), ("fvsr_quantize_fp8", QUANT, dict(cols=0), 1, b"cols"),
    ("fvsr_quantize_fp8", QUANT, dict(rows=1 << 31), 5, b"too large"),
    ("fvsr_quantize_fp8", QUANT, dict(rows=1 << 29, cols=1 << 29), 5, b"too large"),
    ("fvsr_quantize_fp8", QUANT, dict(dtype=2), 1, b"dtype"), ("fvsr_quantize_fp8", QUANT, dict(x=None), 1, b"required"),
    ("fvsr_quantize_fp8", QUANT, dict(q=None), 1, b"together"), ("fvsr_quantize_fp8", QUANT, dict(scale_t=None), 1, b"together"),
    ("fvsr_quantize_fp8", QUANT, dict(q=None, scale=None, qt=None, scale_t=None), 1, b"required"),
    ("fvsr_quantize_fp8", QUANT, dict(x=ODD8), 1, b"aligned"), ("fvsr_quantize_fp8", QUANT, dict(scale_t=ODD8), 1, b"aligned"),
    ("fvsr_fp8_codes", CODES, dict(out=None), 1, b"required"), ("fvsr_fp8_codes", CODES, dict(scale=ODD8), 1, b"aligned"),
    ("fvsr_fp8_codes", CODES, dict(cols=0), 1, b"cols"),
    ("fvsr_dequantize_fp8", DEQUANT, dict(out=None), 1, b"required"), ("fvsr_dequantize_fp8", DEQUANT, dict(out=ODD2), 1, b"aligned"),
    ("fvsr_dequantize_fp8", DEQUANT, dict(q=ODD8), 1, b"aligned"), ("fvsr_dequantize_fp8", DEQUANT, dict(dtype=-1), 1, b"dtype"),
    ("fvsr_linear_fp8", LINEAR, dict(m=-1), 1, b"m must be"), ("fvsr_linear_fp8", LINEAR, dict(n=0), 1, b"n and k"),
    ("fvsr_linear_fp8", LINEAR, dict(k=0), 1, b"n and k"), ("fvsr_linear_fp8", LINEAR, dict(m=(1 << 22) + 1), 5, b"too large"),
    ("fvsr_linear_fp8", LINEAR, dict(m=1 << 21, n=1 << 21), 5, b"too large"),
    ("fvsr_linear_fp8", LINEAR, dict(epilogue=3), 1, b"epilogue"), ("fvsr_linear_fp8", LINEAR, dict(epilogue=-1), 1, b"epilogue"),
    ("fvsr_linear_fp8", LINEAR, dict(x=None), 1, b"required"), ("fvsr_linear_fp8", LINEAR, dict(w_scale=None), 1, b"required"),
    ("fvsr_linear_fp8", LINEAR, dict(gate=None), 1, b"gated"), ("fvsr_linear_fp8", LINEAR, dict(resid=None), 1, b"gated"),
    ("fvsr_linear_fp8", LINEAR, dict(out_dtype=3), 1, b"dtype"), ("fvsr_linear_fp8", LINEAR, dict(x=ODD8), 1, b"aligned"),
    ("fvsr_linear_fp8", LINEAR, dict(w_scale=ODD8), 1, b"aligned"), ("fvsr_linear_fp8", LINEAR, dict(out=ODD2), 1, b"aligned"),
    ("fvsr_linear_fp8", LINEAR, dict(bias=ODD1), 1, b"aligned"), ("fvsr_linear_fp8", LINEAR, dict(resid=ODD2), 1, b"aligned"),
    ("fvsr_linear_fp8", LINEAR, dict(m=500, k=900, x_scale=None, workspace=None), 1, b"workspace"),
    ("fvsr_linear_fp8", LINEAR, dict(m=500, k=900, x_scale=None, workspace_bytes=100), 4, b"workspace"),
    ("fvsr_linear_fp8", LINEAR, dict(m=500, k=900, x_scale=None, workspace=ODD8), 1, b"aligned"),
    ("fvsr_layernorm_train", NORM, dict(m=-1), 1, b"m must"), ("fvsr_layernorm_train", NORM, dict(c=0), 1, b"c >= 1"),
    ("fvsr_layernorm_train", NORM, dict(c=8193), 5, b"8192"), ("fvsr_layernorm_train", NORM, dict(dtype=5), 1, b"dtype"),
    ("fvsr_layernorm_train", NORM, dict(shift=None), 1, b"together"), ("fvsr_layernorm_train", NORM, dict(weight=None), 1, b"together"),
    ("fvsr_layernorm_train", NORM, dict(eps=-1.0), 1, b"eps"), ("fvsr_layernorm_train", NORM, dict(eps=float("nan")), 1, b"eps"),
    ("fvsr_layernorm_train", NORM, dict(rstd=None), 1, b"required"), ("fvsr_layernorm_train", NORM, dict(x=ODD1), 1, b"aligned"),
    ("fvsr_layernorm_train", NORM, dict(dtype=0, scale=ODD2), 1, b"aligned"), ("fvsr_layernorm_train", NORM, dict(mean=ODD2), 1, b"aligned"),
    ("fvsr_layernorm_backward", BACK, dict(bias=None), 1, b"together"), ("fvsr_layernorm_backward", BACK, dict(dx=None), 1, b"required"),
    ("fvsr_layernorm_backward", BACK, dict(x=ODD8), 1, b"aligned"), ("fvsr_layernorm_backward", BACK, dict(dy=ODD1), 1, b"aligned"),
    ("fvsr_layernorm_backward", BACK, dict(dshift=ODD2), 1, b"aligned"), ("fvsr_layernorm_backward", BACK, dict(workspace=None), 1, b"workspace"),
    ("fvsr_layernorm_backward", BACK, dict(workspace_bytes=10), 4, b"workspace"),
    ("fvsr_layernorm_backward", BACK, dict(workspace=ODD8), 1, b"aligned"), ("fvsr_layernorm_backward", BACK, dict(c=9000), 5, b"8192"),
]


@pytest.mark.parametrize("name,good,change,status,words", REFUSED)
def test_refused_on_the_host(fvsr, name, good, change, status, words):
    got, message = _call(fvsr, name, good, **change)
    assert got == status and words in message, (got, message)


def test_nothing_to_do_is_ok(fvsr):
    for name, good, change in (("fvsr_quantize_fp8", QUANT, dict(rows=0)), ("fvsr_dequantize_fp8", DEQUANT, dict(rows=0)),
                               ("fvsr_linear_fp8", LINEAR, dict(m=0)), ("fvsr_layernorm_train", NORM, dict(m=0))):
        assert _call(fvsr, name, good, **change)[0] == fvsr.FVSR_OK


def test_sizes(fvsr):
    v, s = ctypes.c_size_t(), ctypes.c_size_t()
    for rows, cols, want in ((1, 1, (128, 512)), (129, 513, (129 * 640, 2 * 2 * 512)), (0, 5, (0, 0)),
                             (1 << 20, 1 << 20, (1 << 40, (1 << 13) * (1 << 11) * 512))):
        assert fvsr.lib().fvsr_fp8_bytes(rows, cols, ctypes.byref(v), ctypes.byref(s)) == fvsr.FVSR_OK
        assert (v.value, s.value) == want
    assert fvsr.lib().fvsr_fp8_bytes(5, 0, None, None) == fvsr.FVSR_EINVAL
    assert fvsr.lib().fvsr_linear_fp8_workspace_size(5, 6, 7, 1, None) == fvsr.FVSR_EINVAL
    assert fvsr.lib().fvsr_layernorm_backward_workspace_size(5, 6, None) == fvsr.FVSR_EINVAL
    assert fvsr.linear_fp8_workspace_size(0, 6, 7, False) == 0


def test_python_checks_before_the_library(fvsr):
    x = torch.zeros((4, 8))
    for call in (lambda: fvsr.quantize_fp8(x), lambda: fvsr.quantize_fp8(x.double()), lambda: fvsr.layernorm_train(x),
                 lambda: fvsr.layernorm_backward(x, x, x[:, 0], x[:, 0]),
                 lambda: fvsr.linear_fp8(x.bfloat16(), None),
                 lambda: fvsr.Fp8Tensor(x, x, 4, 8),
                 lambda: fvsr.Fp8Tensor(torch.zeros((4, 128), dtype=torch.float8_e4m3fn),
                                        torch.zeros((1, 1, 512), dtype=torch.uint8), 4, 8),
                 lambda: fvsr.Fp8Tensor(torch.zeros((4, 8), dtype=torch.float8_e4m3fn),
                                        torch.zeros((1, 1, 512), dtype=torch.uint8), 4, 8)):
        with pytest.raises(fvsr.FVSRError):
            call()
