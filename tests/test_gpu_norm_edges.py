"""LayerNorm's backward pass on rows whose mean times rstd is beyond fp32's range (constant rows of large values): what stands
beside a row, or past the last one, is no part of any sum."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
import fp8_ref as ref  # noqa: E402
from test_gpu_norm_train import _backward_bars, _case, _placed, _within  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def gpu(fvsr):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return fvsr


@pytest.mark.parametrize("places", [(0, 0, 0), (1, 1, 1), (1, 0, 2)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,c", [(1, 1), (5, 8), (7, 12), (5, 20), (33, 129), (9, 256), (700, 264), (21, 1531), (3, 1536),
                                 (1001, 1536), (7, 4101), (3, 8192)])
def test_constant_rows_of_large_values(gpu, m, c, dtype, places):
    """x = mean = +-2^120 and rstd = 2^9 in the last row and in one between: n is 0 there, -mean * rstd is infinite. Bars as
    in the backward test."""
    x, v, dy, _ = _case(m, c, dtype, True, True, m + c)
    v.pop("shift")
    mean, rstd = x.float().mean(1), torch.ones(m, device="cuda")
    for row, value in ((m // 2, -2.0 ** 120), (m - 1, 2.0 ** 120)):
        x[row], mean[row], rstd[row] = value, value, 512.0
    x8 = gpu.quantize_fp8(x)
    xs, dys = _placed(x, places[0], float("nan"))[1], _placed(dy, places[1], float("inf"))[1]
    for inp, values in ((xs, x), (x8, gpu.dequantize_fp8(x8, dtype=F32))):
        got = gpu.layernorm_backward(dys, inp, mean, rstd, **v, dx=_placed(dy, places[2], 0.0)[1])
        bars = _backward_bars(dy, values, mean, rstd, v)
        for k, t in ref.norm_backward(dy, values, mean, rstd, **v).items():
            _within(got[k], t, bars[k], dtype if k == "dx" else F32)
