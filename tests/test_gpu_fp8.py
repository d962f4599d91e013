"""The 8-bit tensors (quantize_fp8, dequantize_fp8) and the linear layers on them (linear_fp8) against 64-bit references.

Quantising scales by powers of two and rounds once, so values and codes are compared for equality. A linear layer's bar
per element, from its arithmetic: products of two e4m3 values and two powers of two are exact in fp32; the sum over K is
made of at most K additions in fp32, each off by at most 2^-23 of a running sum that is at most S = sum |x w| + |bias|
(an addition that truncates; one that rounds is off by half of that); so |error| <= (K + 8) 2^-23 S before the epilogue. GELU(tanh)'s
slope is below 1.13 and its evaluation is good to 2^-20 of the value; the gate multiplies the error. The output's one
rounding adds half a step, finfo(dtype).eps / 2 of the value."""
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
    return fvsr


def _x(rows, cols, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((rows, cols), generator=g, device="cuda")
    x = x * torch.exp(4.0 * torch.randn((rows, 1), generator=g, device="cuda"))
    return x.to(dtype)


def _same(t, values, codes, cols):
    assert t.shape == tuple(values.shape)
    assert torch.equal(t.codes(), codes)
    fin = torch.isfinite(values).all()
    data = t.data.float()
    if fin:  # stored padding is zero
        assert not data[:, cols:].any()
    scale = torch.exp2(codes.double() - 127).repeat_interleave(128, dim=1)[:, :cols]
    assert torch.equal((data[:, :cols].double() * scale)[torch.isfinite(values)], values[torch.isfinite(values)])
    assert torch.equal(torch.isnan(data[:, :cols]), torch.isnan(values))


SHAPES = [(1, 1), (1, 128), (1, 1536), (2, 129), (127, 127), (128, 512), (129, 513), (777, 1000), (300, 2048), (5, 4100),
          (1000, 8), (640, 640), (1031, 257)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize_is_the_definition(gpu, rows, cols, dtype):
    x = _x(rows, cols, dtype, rows + cols)
    for square in (False, True):
        want, want_t = ref.held(x, square), ref.held(x.t(), square)
        a, b = gpu.quantize_fp8_both(x, square=square)
        _same(a, *want, cols)
        _same(b, *want_t, rows)
        alone, alone_t = gpu.quantize_fp8(x, square=square), gpu.quantize_fp8(x, square=square, transpose=True)
        for got, one in ((a, alone), (b, alone_t)):
            assert torch.equal(got.data.view(torch.uint8), one.data.view(torch.uint8))
            assert torch.equal(got.scale, one.scale)  # the whole tiles, codes beyond the tensor among them
        rt, kt, _ = a.scale.shape
        full = a.scale.view(rt, kt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)
        assert not full[rows:].any() and not full[:, -(-cols // 128):].any()
        for out in (BF16, F32):
            assert torch.equal(gpu.dequantize_fp8(a, dtype=out).double(), want[0].to(out).double())
            assert torch.equal(gpu.dequantize_fp8(b, dtype=out).double(), want_t[0].to(out).double())


def test_quantize_borders_of_the_scale(gpu):
    """Blocks whose largest value is zero, exactly 448 times a power of two, one step above, the smallest and largest
    numbers of the type, subnormals; ties between two e4m3 values."""
    tops = [0.0, 448.0, -448.0, 448.0 * (1 + 2 ** -7), 447.0, 1.75 * 2.0 ** -100, 2.0 ** -126, 2.0 ** -133, 1.5 * 2.0 ** -127,
            2.0 ** 127, 1.75 * 2.0 ** 127, -1.9921875 * 2.0 ** 127, 2.0 ** -118, 1.75 * 2.0 ** -119, 1.7578125 * 2.0 ** -119]
    x = torch.zeros((len(tops), 256), dtype=F32)
    for r, t in enumerate(tops):
        x[r, 5] = t
        x[r, 128:] = t * torch.arange(128) / 256.0
    x = torch.cat([x, torch.full((1, 256), 17.0)])
    x[-1, 0], x[-1, 1:9] = 448.0, torch.tensor([17.0, 19.0, 1.0625, 1.1875, -17.0, 2.0 ** -10, 3 * 2.0 ** -10, 2.0 ** -11])
    for dtype in (BF16, F32):
        y = x.to(dtype).cuda()
        want = ref.held(y)
        _same(gpu.quantize_fp8(y), *want, 256)
        want = ref.held(y.t())
        _same(gpu.quantize_fp8(y, transpose=True), *want, y.shape[0])


@pytest.mark.parametrize("value", [float("inf"), float("-inf"), float("nan")])
def test_a_block_with_an_infinity_or_nan_reads_back_as_nan(gpu, value):
    for dtype in (BF16, F32):
        x = _x(200, 300, dtype, 3)
        x[130, 150] = value
        for square in (False, True):
            a, b = gpu.quantize_fp8_both(x, square=square)
            _same(a, *ref.held(x, square), 300)
            _same(b, *ref.held(x.t(), square), 200)
            back = gpu.dequantize_fp8(a)
            hit = torch.zeros(200, 300, dtype=torch.bool, device="cuda")
            hit[128:200 if square else 131, 128:256] = True
            hit[128:130] &= square
            assert torch.equal(torch.isnan(back), hit)


def _operands(gpu, m, n, k, x_kind, square, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn((m, k), generator=g, device="cuda") * torch.exp(torch.randn((m, 1), generator=g, device="cuda"))
    x = x.to(BF16)
    w8 = gpu.quantize_fp8(torch.randn((n, k), generator=g, device="cuda") / k ** 0.5, square=square)
    xv, wv = ref.held(x)[0], gpu.dequantize_fp8(w8, dtype=F32).double()
    bias = torch.randn((n,), generator=g, device="cuda").to(BF16)
    gate = torch.randn((n,), generator=g, device="cuda").to(BF16)
    return (gpu.quantize_fp8(x) if x_kind == "fp8" else x), w8, xv, wv, bias, gate, g


def _held_to(got, want, size, k, epilogue, gate, dtype):
    err = (k + 8) * 2.0 ** -23 * size
    if epilogue == 1:
        err = 1.13 * err + 2.0 ** -20 * want.abs()
    elif epilogue == 2:
        err = gate.double().abs() * err + 2.0 ** -22 * (want.abs() + gate.double().abs() * size)
    bar = err + torch.finfo(dtype).eps / 2 * (want.abs() + err) + 1e-37
    assert got.dtype == dtype and got.shape == want.shape
    d = (got.double() - want).abs()
    assert (d <= bar).all(), (float((d / bar).max()), float(d.max()))


LINEARS = [(1, 1, 1), (1, 16, 128), (1, 1536, 1536), (1, 77, 1100), (2, 300, 257), (5, 1000, 640), (8, 9216, 1536),
           (16, 129, 4100), (17, 256, 128), (31, 500, 700), (64, 64, 512), (127, 255, 384), (128, 256, 128),
           (129, 257, 129), (200, 1, 1000), (256, 512, 1536), (300, 8, 64), (777, 1000, 1100), (1025, 768, 2500),
           (2048, 1536, 1536), (300, 200, 9000), (1536, 1536, 5000), (2600, 1100, 4700), (2600, 1102, 8300), (4000, 1604, 300), (300, 301, 4000)]


@pytest.mark.parametrize("m,n,k", LINEARS)
def test_linear_fp8_against_64_bits(gpu, m, n, k):
    for i, (x_kind, square, dtype, epilogue, biased) in enumerate([
            ("bf16", True, BF16, 0, True), ("fp8", False, F32, 0, False), ("bf16", False, F32, 1, True),
            ("fp8", True, BF16, 1, False), ("fp8", False, BF16, 2, True), ("bf16", True, F32, 2, False)]):
        x, w8, xv, wv, bias, gate, g = _operands(gpu, m, n, k, x_kind, square, 7 * i + m + n + k)
        resid = torch.randn((m, n), generator=g, device="cuda").to(dtype) if epilogue == 2 else None
        got = gpu.linear_fp8(x, w8, bias if biased else None, epilogue=epilogue, gate=gate if epilogue == 2 else None,
                             resid=resid, out_dtype=dtype)
        want, size = ref.linear(xv, wv, bias if biased else None, epilogue, gate, resid)
        _held_to(got, want, size, k, epilogue, gate, dtype)
    gpu.device_check()


@pytest.mark.parametrize("m,n,k", [(1, 300, 700), (9, 300, 700), (40, 300, 700), (500, 300, 700), (130, 256, 9000)])
def test_linear_fp8_forms_agree_and_repeat(gpu, m, n, k):
    """bf16 input and its 8-bit form give the same bits; so does a second call; resid may be out; a given workspace and
    out are used, and nothing beyond out's end is written."""
    x, w8, _, _, bias, gate, g = _operands(gpu, m, n, k, "bf16", True, 11)
    a, b = gpu.linear_fp8(x, w8, bias), gpu.linear_fp8(gpu.quantize_fp8(x), w8, bias)
    assert torch.equal(a, b) and torch.equal(a, gpu.linear_fp8(x, w8, bias))
    resid = torch.randn((m, n), generator=g, device="cuda").to(BF16)
    want = gpu.linear_fp8(x, w8, bias, epilogue=2, gate=gate, resid=resid)
    room = torch.full((m * n + 64,), 7.0, dtype=BF16, device="cuda")
    out = room[:m * n].view(m, n)
    out.copy_(resid)
    need = gpu.linear_fp8_workspace_size(m, n, k, False)
    ws = torch.full((need + 64,), 0xA5, dtype=torch.uint8, device="cuda")
    assert gpu.linear_fp8(x, w8, bias, epilogue=2, gate=gate, resid=out, out=out, workspace=ws[:need]) is not None
    assert torch.equal(out, want) and (room[m * n:] == 7.0).all() and (ws[need:] == 0xA5).all()
    gpu.device_check()


@pytest.mark.parametrize("m,n,k", [(5, 128, 256), (300, 512, 640), (2600, 1104, 8300)])
def test_linear_fp8_into_an_output_off_the_16_byte_grid(gpu, m, n, k):
    """out and resid that start two or four bytes past the grid are written element by element: the same bits."""
    for dtype in (BF16, F32):
        x, w8, _, _, bias, gate, g = _operands(gpu, m, n, k, "fp8", True, 5)
        resid = torch.randn((m, n), generator=g, device="cuda").to(dtype)
        want = gpu.linear_fp8(x, w8, bias, epilogue=2, gate=gate, resid=resid, out_dtype=dtype)
        off = 2 if dtype == BF16 else 1
        room, held = (torch.full((m * n + 64,), 7.0, dtype=dtype, device="cuda") for _ in range(2))
        out, res = room[off:off + m * n].view(m, n), held[off:off + m * n].view(m, n)
        res.copy_(resid)
        gpu.linear_fp8(x, w8, bias, epilogue=2, gate=gate, resid=res, out=out)
        assert torch.equal(out, want)
        assert (room[:off] == 7.0).all() and (room[off + m * n:] == 7.0).all()
    gpu.device_check()


def test_host_threads_on_streams_of_their_own(gpu):
    """Four host threads, each with a stream and operands of its own, at once: each gets what a call alone gives."""
    import threading
    jobs = [_operands(gpu, m, 700, 1500, "bf16", True, 50 + m)[:2] for m in (1, 40, 300, 600)]
    want = [gpu.linear_fp8(*j) for j in jobs]
    torch.cuda.synchronize()
    errors = []

    def work(i):
        try:
            st = torch.cuda.Stream()
            got = [gpu.linear_fp8(*jobs[i], stream=st) for _ in range(20)]
            st.synchronize()
            assert all(torch.equal(t, want[i]) for t in got)
        except BaseException as e:  # re-raised below
            errors.append(e)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in ts:
        t.start()
    for t in ts:
        t.join(60)
    assert not errors, errors
    gpu.device_check()


def test_linear_fp8_accuracy_of_a_long_sum(gpu):
    """fp32 sums over a long K stay fp32: relative to the result's norm, K = 17280 random products summed in fp32 are
    off by about sqrt(K) roundings of the running sum at worst, sqrt(17280) 2^-24 = 8e-6; twice that is the bar (an
    accumulator of 14 or 22 bits would be off by 1e-3 or 4e-5)."""
    x8, w8 = (gpu.quantize_fp8(_x(400, 17280, F32, s) / 50) for s in (1, 2))
    xv, wv = (gpu.dequantize_fp8(t, dtype=F32).double() for t in (x8, w8))
    got = gpu.linear_fp8(x8, w8, out_dtype=F32).double()
    want = xv @ wv.t()
    rows = ((got - want).norm(dim=1) / want.norm(dim=1)).max()
    assert rows <= 2 * 17280 ** 0.5 * 2.0 ** -24, float(rows)


def test_linear_fp8_of_a_nan_block_is_nan_there_only(gpu):
    for m in (3, 200):
        x = _x(m, 600, BF16, 5)
        x[2, 300] = float("nan")
        w8 = gpu.quantize_fp8(_x(260, 600, BF16, 6), square=True)
        for inp in (x, gpu.quantize_fp8(x)):
            y = gpu.linear_fp8(inp, w8)
            nan = torch.isnan(y)
            assert nan[2].all() and not nan[:2].any() and not nan[3:].any()


def test_empty_and_zero(gpu):
    w8 = gpu.quantize_fp8(torch.zeros((70, 200), device="cuda"))
    assert not gpu.dequantize_fp8(w8).any()
    assert gpu.linear_fp8(torch.empty((0, 200), dtype=BF16, device="cuda"), w8).shape == (0, 70)
    assert not gpu.linear_fp8(torch.ones((20, 200), dtype=BF16, device="cuda"), w8).any()
    e = gpu.quantize_fp8(torch.empty((0, 9), device="cuda"))
    assert e.shape == (0, 9) and gpu.dequantize_fp8(e).shape == (0, 9)


@pytest.mark.parametrize("m,n,k", [(1, 512, 1536), (300, 520, 1000), (256, 256, 8192)])
def test_linear_fp8_on_a_side_stream_and_in_a_graph(gpu, m, n, k):
    x, w8, _, _, bias, _, g = _operands(gpu, m, n, k, "bf16", True, 21)
    want = gpu.linear_fp8(x, w8, bias)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = [gpu.linear_fp8(x, w8, bias, stream=side) for _ in range(3)]
    side.synchronize()
    assert all(torch.equal(t, want) for t in got)
    x2 = torch.randn((m, k), generator=g, device="cuda").to(BF16)
    want2 = gpu.linear_fp8(x2, w8, bias)
    gr, hold = torch.cuda.CUDAGraph(), x.clone()
    with torch.cuda.graph(gr):
        q, qt = gpu.quantize_fp8_both(hold)
        out, out8 = gpu.linear_fp8(hold, w8, bias), gpu.linear_fp8(q, w8, bias)
    for src, res in ((x, want), (x2, want2), (x, want)):
        hold.copy_(src)
        gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, res) and torch.equal(out8, res)
    gpu.device_check()


def test_two_streams_at_once(gpu):
    """Two calls in flight on two streams, each with a workspace of its own, give what each gives alone."""
    jobs = [_operands(gpu, 400 + 100 * i, 1536, 4000, "bf16", True, 31 + i)[:2] for i in range(2)]
    want = [gpu.linear_fp8(*j) for j in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(4):
        for i in range(2):
            got[i].append(gpu.linear_fp8(*jobs[i], stream=streams[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(t, want[i]) for t in got[i])
    gpu.device_check()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("rows,cols", [(1, 1), (3, 5), (4, 8), (5, 127), (7, 131), (9, 511), (6, 513), (3, 1531), (2, 1536)])
def test_dequantize_into_an_output_at_any_offset(gpu, rows, cols, dtype):
    x8 = gpu.quantize_fp8(_x(rows, cols, dtype, rows + cols))
    want = gpu.dequantize_fp8(x8, dtype=F32).to(dtype)
    for off in range(9):
        room = torch.full((rows * cols + 32,), 3.0, dtype=dtype, device="cuda")
        out = room[8 + off:8 + off + rows * cols].view(rows, cols)
        if out.data_ptr() % 4:
            with pytest.raises(gpu.FVSRError, match="aligned"):
                gpu.dequantize_fp8(x8, dtype=dtype, out=out)
            continue
        gpu.dequantize_fp8(x8, dtype=dtype, out=out)
        assert torch.equal(out, want)
        assert (room[:8 + off] == 3.0).all() and (room[8 + off + rows * cols:] == 3.0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,n,k", [(17, 1, 40), (40, 7, 130), (300, 129, 64), (257, 515, 200)])
def test_a_residual_between_values_that_are_not_its_own(gpu, m, n, k, dtype):
    """NaN before and behind a residual at each offset from the 16-byte grid that it may have (whole 4 bytes; others are
    refused): the bits that it gives on the grid."""
    g = torch.Generator(device="cuda").manual_seed(m + n)
    x8, w8 = gpu.quantize_fp8(_x(m, k, BF16, 1)), gpu.quantize_fp8(_x(n, k, BF16, 2))
    gate = torch.randn(n, generator=g, device="cuda").to(BF16)
    resid = torch.randn((m, n), generator=g, device="cuda").to(dtype)
    want = gpu.linear_fp8(x8, w8, epilogue=2, gate=gate, resid=resid, out_dtype=dtype)
    assert torch.isfinite(want).all()
    for off in (0, 1, 2, 4, 6) if dtype == BF16 else (0, 1, 3):
        room = torch.full((m * n + 32,), float("nan"), dtype=dtype, device="cuda")
        res = room[8 + off:8 + off + m * n].view(m, n)
        res.copy_(resid)
        if res.data_ptr() % 4:
            with pytest.raises(gpu.FVSRError, match="aligned"):
                gpu.linear_fp8(x8, w8, epilogue=2, gate=gate, resid=res, out_dtype=dtype)
            continue
        assert torch.equal(gpu.linear_fp8(x8, w8, epilogue=2, gate=gate, resid=res, out_dtype=dtype), want)
