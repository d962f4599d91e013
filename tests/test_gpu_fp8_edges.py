"""The 8-bit linear layers where their arithmetic or their reach ends: what a workspace held before, scales at the ends of
fp32's range, long sums, sizes beyond 32 bits, temporaries of a call on another stream."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
import fp8_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def gpu(fvsr):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    yield fvsr
    torch.cuda.empty_cache()


def _rand(seed, *shape):
    return torch.randn(shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [(300, 301, 4000), (40, 1, 4000), (64, 515, 2100), (300, 302, 4000)])
def test_a_sum_in_parts_does_not_depend_on_what_the_workspace_held(gpu, m, n, k, dtype):
    """GELU shares a reciprocal between neighbouring columns, and the planes of partial sums have rows of a multiple of four:
    an odd last column must not have its neighbour from memory that nothing wrote."""
    x8, w8 = gpu.quantize_fp8(_rand(1, m, k)), gpu.quantize_fp8(_rand(2, n, k) / k ** 0.5)
    need = gpu.linear_fp8_workspace_size(m, n, k, True)
    ld = -(-n // 4) * 4
    assert need >= 2 * m * ld * 4  # in parts
    got = []
    for fill in (0x00, 0x3D, 0x3E, 0xBE, 0x7F, 0xC2, 0xFF):  # 0, 0.046, 0.19, -0.37, 3.4e38, -97, NaN
        ws = torch.full((need,), fill, dtype=torch.uint8, device="cuda")
        got.append(gpu.linear_fp8(x8, w8, epilogue=1, out_dtype=dtype, workspace=ws))
        sums = ws.view(F32)[:need // 4 // (m * ld) * m * ld].view(-1, m, ld)
        assert not sums[:, :, n:].any()
    assert torch.isfinite(got[0]).all()
    assert all(torch.equal(t, got[0]) for t in got[1:])
    gpu.device_check()
