"""The 8-bit linear layers where their arithmetic or their reach ends: what a workspace held before, scales at the ends of
fp32's range, long sums, sizes beyond 32 bits, temporaries of a call on another stream."""
from __future__ import annotations

import math

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


@pytest.mark.parametrize("m", [1, 9, 16, 17, 40, 300])
def test_scales_that_meet_beyond_the_range_of_fp32(gpu, m):
    """Operands of 2^118 and 2^-118: their products are ordinary numbers, their scales and the sums before scaling are not.
    Bar: the sum's additions as in the linear layers' tests, (K + 8) 2^-23 sum|x w|, and the rounding of the output."""
    n = 70
    for k in (128, 700):
        for e in (-118, -60, 60, 118):
            x = (_rand(m + k, m, k) * 2.0 ** e).to(BF16)
            x8, w8 = gpu.quantize_fp8(x), gpu.quantize_fp8(_rand(k, n, k) * 2.0 ** -e)
            want, size = ref.linear(*(gpu.dequantize_fp8(t, dtype=F32).double() for t in (x8, w8)))
            bar = (k + 8) * 2.0 ** -23 * size + 2.0 ** -24 * want.abs()
            for inp in (x, x8):
                d = (gpu.linear_fp8(inp, w8, out_dtype=F32).double() - want).abs()
                assert (d <= bar).all(), (k, e, float((d / bar).max()))
    gpu.device_check()


def test_rows_and_channels_beyond_32_bits_are_refused(gpu):
    """Not taken modulo 2^32, which gave the first 5 rows, or the statistics of the first 8 channels."""
    rows = (1 << 32) + 5
    x = torch.empty((rows, 1), dtype=BF16, device="cuda")
    w8 = gpu.quantize_fp8(torch.ones((1, 1), device="cuda"))
    with pytest.raises(gpu.FVSRError, match="too large"):
        gpu.linear_fp8(x, w8)
    x = x.view(-1)[:(1 << 32)].view(1, -1)
    stat = torch.ones(1, device="cuda")
    with pytest.raises(gpu.FVSRError, match="too large"):
        gpu.layernorm_train(x)
    with pytest.raises(gpu.FVSRError, match="too large"):
        gpu.layernorm_backward(x, x, stat, stat)


def test_temporaries_of_a_call_on_another_stream(gpu):
    """Inputs that the caller lets go after a call on a stream that has not run yet: their memory is not given to the next
    allocation of their own stream."""
    x = _rand(1, 400, 512).to(BF16)
    w8, v = gpu.quantize_fp8(_rand(2, 300, 512)), _rand(3, 512).to(BF16)
    out, mean, rstd = gpu.layernorm_train(x, shift=v, scale=v)
    calls = [
        (lambda s, t: gpu.linear_fp8(t, w8, stream=s), lambda: x.clone()),
        (lambda s, t: gpu.linear_fp8(t, w8, stream=s), lambda: gpu.quantize_fp8(x)),
        (lambda s, t: gpu.linear_fp8(x, t, stream=s), lambda: gpu.quantize_fp8(_rand(2, 300, 512))),
        (lambda s, t: gpu.quantize_fp8(t, stream=s).codes(), lambda: x.clone()),
        (lambda s, t: gpu.dequantize_fp8(t, stream=s), lambda: gpu.quantize_fp8(x)),
        (lambda s, t: gpu.layernorm_train(t, shift=v, scale=v, stream=s)[0], lambda: x.clone()),
        (lambda s, t: gpu.layernorm_backward(t, x, mean, rstd, stream=s)["dx"], lambda: x.clone()),
        (lambda s, t: gpu.layernorm_backward(x, t, mean, rstd, stream=s)["dx"], lambda: gpu.quantize_fp8(x)),
    ]
    side = torch.cuda.Stream()
    for i, (call, make) in enumerate(calls):
        want = call(None, make())
        torch.cuda.synchronize()
        t = make()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
        if i == 3:  # the codes are of the 8-bit tensor that the side stream fills
            held = gpu.quantize_fp8(t, stream=side)
            got = None
        else:
            got = call(side, t)
        del t
        junk = [torch.full((400, 512), float("nan"), device="cuda", dtype=BF16) for _ in range(4)]
        junk += [torch.full((n, 512), 255, device="cuda", dtype=torch.uint8) for n in (400, 300, 400, 300, 4, 3, 4, 3)]
        torch.cuda.synchronize()
        got = held.codes() if got is None else got
        assert torch.equal(got, want), i
        del junk
    gpu.device_check()


def _products(gpu, m, n, k, one_sign):
    """8-bit operands (m, k), (n, k) of random values, or of their magnitudes, and their product in 64 bits."""
    x, w = _rand(m + k, m, k), _rand(n + k + 1, n, k)
    x8, w8 = gpu.quantize_fp8(x.abs_() if one_sign else x), gpu.quantize_fp8(w.abs_() if one_sign else w)
    xv, wv = (gpu.dequantize_fp8(t, dtype=F32, out=o) for t, o in ((x8, x), (w8, w)))
    want = torch.zeros((m, n), dtype=torch.float64, device="cuda")
    for at in range(0, k, 1 << 15):
        want += xv[:, at:at + (1 << 15)].double() @ wv[:, at:at + (1 << 15)].double().t()
    return x8, w8, want


# An addition of 32 products truncates by at most 2^-23 of the running sum, which products of one sign let grow evenly: a chain
# of c additions is off by at most (c + 1) / 2 * 2^-23 of its sum. In chains of 4096 (c = 128) that is 64.5 * 2^-23 = 7.7e-6,
# and each addition of chains rounds by half of that step; one chain of 17280 was measured at 1.1e-5.
SIGNED = 64.5 * 2.0 ** -23
LONG = [(1280, 2048, 17280), (1280, 2046, 17280), (1280, 2047, 17280),  # not cut: chains in the output, on and off the grid
        (1536, 1536, 34560), (1280, 1533, 34560)]                        # in two parts: chains in the planes of partial sums


@pytest.mark.parametrize("m,n,k", LONG)
def test_long_fp32_sums_are_taken_in_chains(gpu, m, n, k):
    """One sign: each value within the bar above. Zero mean: relative to the result's norm, a chain of 4096 was measured at
    2.2e-7 and one of 17280 at 1.3e-6; 6e-7 tells them apart."""
    x8, w8, want = _products(gpu, m, n, k, True)
    got = gpu.linear_fp8(x8, w8, out_dtype=F32).double()
    bar = SIGNED + (k // 4096 + 2) * 2.0 ** -24
    assert float(((got - want).abs() / want).max()) <= bar
    # in place, gated: resid + gate * (x w), the gate a power of two, the residual about the sum's size
    gate = torch.full((n,), 0.5, dtype=BF16, device="cuda")
    resid = want.to(F32).clone()
    start = resid.double() + 0.5 * want
    out = gpu.linear_fp8(x8, w8, epilogue=2, gate=gate, resid=resid, out=resid)
    assert out.data_ptr() == resid.data_ptr()
    assert float(((out.double() - start).abs() / start).max()) <= bar + (k // 4096 + 2) * 2.0 ** -24
    x8, w8, want = _products(gpu, m, n, k, False)
    got = gpu.linear_fp8(x8, w8, out_dtype=F32).double()
    assert float(((got - want).norm(dim=1) / want.norm(dim=1)).max()) <= 6e-7
    gpu.device_check()


@pytest.mark.parametrize("m,n,k", [(1280, 2048, 1 << 18), (1280, 2047, 70000), (300, 301, 1 << 18), (20, 33, 1 << 22)])
def test_long_bf16_sums(gpu, m, n, k):
    """A bf16 output's chains end at 65536 (c = 2048 additions: (c + 1) / 2 * 2^-23 = 1.22e-4; one chain of 2^18 was measured
    at 4.2e-4). A residual that cancels the sum shows its error; what is left is rounded to bf16."""
    x8, w8, want = _products(gpu, m, n, k, True)
    resid = (-want).to(BF16)
    one = torch.ones((n,), dtype=BF16, device="cuda")
    left = want + resid.double()
    err = (1024.5 * 2.0 ** -23 + (k // 65536 + 70) * 2.0 ** -24) * want  # up to 70 parts are added up
    for fill in (0x00, 0xFF):
        ws = torch.full((gpu.linear_fp8_workspace_size(m, n, k, True),), fill, dtype=torch.uint8, device="cuda")
        got = gpu.linear_fp8(x8, w8, epilogue=2, gate=one, resid=resid, workspace=ws)
        assert ((got.double() - left).abs() <= err + 2.0 ** -8 * (left.abs() + err)).all()
    got = gpu.linear_fp8(x8, w8)
    assert ((got.double() - want).abs() <= err + 2.0 ** -8 * (want + err)).all()
    gpu.device_check()


def test_a_forked_stream_in_a_captured_graph(gpu):
    """The same inside a capture that forks to a second stream: replays give what the calls give."""
    w8, v = gpu.quantize_fp8(_rand(2, 300, 512)), _rand(3, 512).to(BF16)
    hold = _rand(1, 400, 512).to(BF16)
    side = torch.cuda.Stream()

    def step(fork):
        s = None
        q = gpu.quantize_fp8(hold)
        if fork:
            s = side
            side.wait_stream(torch.cuda.current_stream())
        y = gpu.linear_fp8(q, w8, stream=s)
        n = gpu.layernorm_train(hold, shift=v, scale=v, stream=s)
        del q
        back = [gpu.quantize_fp8(hold * i) for i in (2.0, 3.0)]  # of the freed size, on the first stream
        if fork:
            torch.cuda.current_stream().wait_stream(side)
        return [y, *n] + [gpu.dequantize_fp8(b) for b in back]

    step(False)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step(True)
    for seed in (4, 5):
        hold.copy_(_rand(seed, 400, 512))
        want = step(False)
        for _ in range(3):
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, want))
    gpu.device_check()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [(3, 24, 128), (16, 64, 300), (40, 64, 256), (300, 64, 4000)])
def test_gelu_of_large_values(gpu, m, n, k, dtype):
    """GELU beside values of any size: below -7.45, where its exact value is between -1e-17 and 0, nothing but that; the value
    itself where it is large; NaN alone. Bar of the ordinary columns between them: as in the linear layers' tests."""
    x8, w8 = gpu.quantize_fp8(_rand(1, m, k)), gpu.quantize_fp8(_rand(2, n, k) / k ** 0.5)
    bias = _rand(3, n).to(BF16)
    large = torch.tensor([-20.0, -1e4, -1e20, -3e38, 20.0, 1e4, 1e20, 3e38], device="cuda").to(BF16)
    bias[1::8] = large[:n // 8]
    bias[6::8] = float("nan")
    got = gpu.linear_fp8(x8, w8, bias, epilogue=1, out_dtype=dtype).double()
    y, size = ref.linear(*(gpu.dequantize_fp8(t, dtype=F32).double() for t in (x8, w8)), bias)
    want = torch.where(y.abs() > 30, y.clamp(min=0.0), y / (1.0 + torch.exp(-2.0 * (2.0 / math.pi) ** 0.5 * (y + 0.044715 * y ** 3))))
    cols = torch.arange(n, device="cuda")
    assert got[:, cols % 8 == 6].isnan().all() and not got[:, cols % 8 != 6].isnan().any()
    far = (y < -7.45) & ~y.isnan()
    assert far.any() and (got[far].abs() <= 1.01e-17).all()
    near = ~far & ~y.isnan()
    bar = 1.13 * (k + 8) * 2.0 ** -23 * size + 2.0 ** -20 * want.abs()
    bar = bar + torch.finfo(dtype).eps / 2 * (want.abs() + bar)
    assert ((got - want).abs() <= bar)[near].all()
    gpu.device_check()
