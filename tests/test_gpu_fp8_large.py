"""Tensors of more than 2^32 elements: every offset of the 8-bit tensors, the linear layers on them and LayerNorm's training
passes is formed in 64 bits. The rows at the far end must come out as the same rows alone do (each row, and each block of
128 rows of a transposed form, is computed on its own, so the bits are equal)."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def gpu(fvsr):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    if torch.cuda.get_device_properties(0).total_memory < 120 << 30:
        pytest.skip("needs 120 GB")
    yield fvsr
    torch.cuda.empty_cache()


def _tall(rows, cols, tail, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.zeros((rows, cols), dtype=BF16, device="cuda")
    x[-tail:] = torch.randn((tail, cols), generator=g, device="cuda").to(BF16)
    return x


def test_quantize_and_back(gpu):
    rows, cols, tail = 128 * 8300 + 3, 4104, 259   # 4.36e9 elements; the tail starts at a block of 128 rows
    x = _tall(rows, cols, tail, 1)
    end = x[-tail:].clone()
    a, b = gpu.quantize_fp8_both(x)
    ea, eb = gpu.quantize_fp8_both(end)
    assert torch.equal(a.data[-tail:].view(torch.uint8), ea.data.view(torch.uint8))
    assert torch.equal(b.data[:, rows - tail:rows].float(), eb.data[:, :tail].float())
    assert torch.equal(a.codes()[-tail:], ea.codes()) and torch.equal(b.codes()[:, -3:], eb.codes())
    assert not a.data[:rows - tail].view(torch.uint8).any()
    del b, x
    assert torch.equal(gpu.dequantize_fp8(a)[-tail:], gpu.dequantize_fp8(ea))


def test_norms(gpu):
    rows, cols, tail = 128 * 8300 + 3, 4104, 259
    x = _tall(rows, cols, tail, 2)
    end = x[-tail:].clone()
    v = torch.linspace(-1, 1, cols, device="cuda").to(BF16)
    out, mean, rstd = gpu.layernorm_train(x, shift=v, scale=v)
    want = gpu.layernorm_train(end, shift=v, scale=v)
    assert torch.equal(out[-tail:], want[0]) and torch.equal(mean[-tail:], want[1]) and torch.equal(rstd[-tail:], want[2])
    for held in (False, True):
        inp, one = (gpu.quantize_fp8(x), gpu.quantize_fp8(end)) if held else (x, end)
        dx = gpu.layernorm_backward(out, inp, mean, rstd, scale=v)["dx"]
        assert torch.equal(dx[-tail:], gpu.layernorm_backward(want[0], one, want[1], want[2], scale=v)["dx"])
        del dx, inp


@pytest.mark.parametrize("n", [8192, 8191])
def test_linear(gpu, n):
    rows, k, tail = 256 * 2100 + 5, 128, 517       # 4.4e9 outputs
    x = _tall(rows, k, tail, 3)
    end = x[-tail:].clone()
    w8 = gpu.quantize_fp8(torch.randn((n, k), device="cuda"), square=True)
    bias = torch.randn((n,), device="cuda").to(BF16)
    out = gpu.linear_fp8(x, w8, bias)
    assert torch.equal(out[-tail:], gpu.linear_fp8(end, w8, bias))
    assert torch.equal(out[5], bias)
    gpu.device_check()
