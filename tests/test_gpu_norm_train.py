"""LayerNorm for training (layernorm_train, layernorm_backward) against 64-bit references, and a training step of norm
and linear layer in 8 bits as a whole.

Bars, with u = 2^-24 (half a step of fp32) and sums that add at most d values one after another in any thread (d <= 80:
8192 channels over at least 128 threads, or 64 to a lane, and the tree above them):
  mean         d u mean|x|
  n            e_n = rstd (d u mean|x| + 2u |x - mean|) + (d + 8) u |n|   (rstd: half the variance's relative error)
  y            |w (1 + scale)| e_n + 4u (|n w (1 + scale)| + |b (1 + scale)| + |shift|)
  dx           its terms, each with the error of what it is made of (below), n here from the given mean and rstd
  vector sums  (rows + 8) u sum|terms| and the terms' own errors
and half a step of the output's type for its one rounding."""
from __future__ import annotations

import pytest

torch = pytest.importorskip("torch")
import fp8_ref as ref  # noqa: E402

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
U, D = 2.0 ** -24, 80


@pytest.fixture(scope="module")
def gpu(fvsr):
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")
    return fvsr


def _case(m, c, dtype, affine, modulated, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def r(*shape, base=0.0, size=1.0):
        return (base + size * torch.randn(shape, generator=g, device="cuda")).to(dtype)

    x = (torch.randn((m, c), generator=g, device="cuda") * 1.5 + torch.randn((m, 1), generator=g, device="cuda")).to(dtype)
    v = {"weight": r(c, base=1.0, size=0.2), "bias": r(c, size=0.3)} if affine else {"weight": None, "bias": None}
    v |= {"shift": r(c, size=0.3), "scale": r(c, size=0.3)} if modulated else {"shift": None, "scale": None}
    return x, v, r(m, c, size=1e-2), g


def _vec(v, like):
    one = torch.ones(like.shape[1], dtype=torch.float64, device=like.device)
    d = {k: (t.double() if t is not None else None) for k, t in v.items()}
    return (d["weight"] if d["weight"] is not None else one, d["bias"] if d["bias"] is not None else 0 * one,
            1.0 + d["scale"] if d.get("scale") is not None else one, d["shift"] if d.get("shift") is not None else 0 * one)


def _within(got, want, err, dtype=F32):
    bar = err + torch.finfo(dtype).eps / 2 * (want.abs() + err) + 1e-37
    d = (got.double() - want).abs()
    assert got.dtype == dtype and got.shape == want.shape
    assert (d <= bar).all(), (float((d / bar).max()), float(d.max()))


SHAPES = [(1, 1), (1, 1536), (3, 2), (7, 8), (1, 8192), (5, 8191), (300, 129), (777, 1000), (129, 256), (600, 1536),
          (64, 2048), (33, 4096), (1200, 100), (2000, 512), (50, 2056), (100, 1030)]


@pytest.mark.parametrize("affine,modulated", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,c", SHAPES)
def test_forward(gpu, m, c, dtype, affine, modulated):
    x, v, _, _ = _case(m, c, dtype, affine, modulated, m + c)
    out, mean, rstd = gpu.layernorm_train(x, **v)
    want, mean_w, rstd_w = ref.norm(x, **v)
    xd = x.double()
    size = xd.abs().mean(1)
    _within(mean, mean_w, D * U * size)
    n = (xd - mean_w[:, None]) * rstd_w[:, None]
    # a variance about a mean that is off by e is off by e^2 more: relative to var + eps, (rstd D U size)^2
    rel = (D + 8) * U + (rstd_w * D * U * size) ** 2
    _within(rstd, rstd_w, rel * rstd_w)
    e_n = rstd_w[:, None] * (D * U * size[:, None] + 2 * U * (xd - mean_w[:, None]).abs()) + rel[:, None] * n.abs()
    w, b, s1, sh = _vec(v, x)
    _within(out, want, (w * s1).abs() * e_n + 4 * U * ((n * w * s1).abs() + (b * s1).abs() + sh.abs()), dtype)
    again = gpu.layernorm_train(x, **v, out=x)
    assert torch.equal(again[0], out) and again[0].data_ptr() == x.data_ptr()


def _backward_bars(dy, x, mean, rstd, v):
    w, b, s1, _ = _vec(v, x)
    dy, x, mean, rstd = dy.double(), x.double(), mean.double()[:, None], rstd.double()[:, None]
    n = (x - mean) * rstd
    e_n = U * (rstd * (x - mean).abs() + 2 * n.abs())
    g = dy * s1 * w
    e_g = 4 * U * g.abs()
    e1 = (D * U * g.abs() + e_g).mean(1, keepdim=True)
    m2 = (g * n).mean(1, keepdim=True)
    e2 = (D * U * (g * n).abs() + e_g * n.abs() + g.abs() * e_n).mean(1, keepdim=True)
    e_dx = rstd * (e_g + e1 + n.abs() * e2 + m2.abs() * e_n
                   + 4 * U * (g.abs() + g.mean(1, keepdim=True).abs() + (n * m2).abs()))
    rows = dy.shape[0]
    e_a = ((rows + 8) * U * (dy * n).abs() + dy.abs() * e_n).sum(0)
    e_b = ((rows + 8) * U * dy.abs()).sum(0)
    a, s = (dy * n).sum(0).abs(), dy.sum(0).abs()
    return {"dx": e_dx, "dweight": s1.abs() * (e_a + 2 * U * a), "dbias": s1.abs() * (e_b + 2 * U * s),
            "dscale": w.abs() * (e_a + 2 * U * a) + b.abs() * (e_b + 2 * U * s), "dshift": e_b}


@pytest.mark.parametrize("affine,modulated", [(False, False), (True, False), (False, True), (True, True)])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,c", SHAPES)
def test_backward(gpu, m, c, dtype, affine, modulated):
    x, v, dy, _ = _case(m, c, dtype, affine, modulated, m + c + 1)
    _, mean, rstd = gpu.layernorm_train(x, **v)
    v.pop("shift")
    x8 = gpu.quantize_fp8(x)
    for inp, values in ((x, x), (x8, gpu.dequantize_fp8(x8, dtype=F32))):
        got = gpu.layernorm_backward(dy, inp, mean, rstd, **v)
        want = ref.norm_backward(dy, values, mean, rstd, **v)
        bars = _backward_bars(dy, values, mean, rstd, v)
        for k, t in want.items():
            assert (got[k] is None) == (t is None)
            if t is not None:
                _within(got[k], t, bars[k], dtype if k == "dx" else F32)
        again = gpu.layernorm_backward(dy, inp, mean, rstd, **v, dx=dy.clone())
        assert all(got[k] is None or torch.equal(got[k], again[k]) for k in got)
        held = dy.clone()
        gpu.layernorm_backward(held, inp, mean, rstd, **v, dx=held)
        assert torch.equal(held, got["dx"])


def test_backward_against_differences(gpu):
    """The gradients along random directions against central differences of the 64-bit forward pass. With step h the
    difference is off by h^2 / 6 of the third derivative (order 1 here, h = 1e-4) and 2^-52 / h of the value; the kernel's
    own error is fp32's: bar 1e-5 of the sum of the terms' magnitudes."""
    x, v, dy, g = _case(40, 200, F32, True, True, 5)
    _, mean, rstd = gpu.layernorm_train(x, **v)
    got = gpu.layernorm_backward(dy, x, mean, rstd, weight=v["weight"], bias=v["bias"], scale=v["scale"])
    xs = {"x": x.double(), **{k: t.double() for k, t in v.items()}}
    names = {"x": "dx", "weight": "dweight", "bias": "dbias", "shift": "dshift", "scale": "dscale"}
    for k, grad in names.items():
        way = torch.randn(xs[k].shape, generator=g, device="cuda", dtype=torch.float64)
        h, val = 1e-4, []
        for sign in (1, -1):
            args = dict(xs)
            args[k] = xs[k] + sign * h * way
            val.append((ref.norm(**args)[0] * dy.double()).sum())
        diff, mine = (val[0] - val[1]) / (2 * h), (got[grad].double() * way).sum()
        assert abs(diff - mine) <= 1e-5 * (got[grad].double() * way).abs().sum(), (k, float(diff), float(mine))


def test_rows_without_spread_and_bad_rows(gpu):
    """A constant row: n = 0, so y is the bias chain and rstd 1 / sqrt(eps); eps = 0 gives infinity and NaN there as the
    formula does. A row with a NaN or an infinity is NaN, its neighbours are not touched."""
    for c in (256, 77):
        x = torch.randn((6, c), device="cuda", dtype=F32)
        x[1] = 0.25
        x[3, 5] = float("nan")
        x[4, 7] = float("inf")
        out, mean, rstd = gpu.layernorm_train(x, eps=1e-6)
        assert (out[1] == 0).all() and abs(float(rstd[1]) - 1e3) <= 1e3 * 4 * U + 1e-4
        assert torch.isnan(out[3:5]).all() and not torch.isnan(out[[0, 1, 2, 5]]).any()
        dy = torch.randn_like(x)
        dx = gpu.layernorm_backward(dy, x, mean, rstd)["dx"]
        assert torch.isnan(dx[3:5]).all() and torch.isfinite(dx[[0, 1, 2, 5]]).all()
        assert torch.isnan(gpu.layernorm_train(x, eps=0.0)[0][1]).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("c", [256, 1536, 1000])
def test_tensors_off_the_16_byte_grid(gpu, c, dtype):
    """Contiguous views that start one element into a buffer: the same values as aligned tensors, nothing written outside."""
    m = 70
    x, v, dy, _ = _case(m, c, dtype, True, True, 3)

    def shifted(t):
        room = torch.full((t.numel() + 2,), 3.0, dtype=t.dtype, device="cuda")
        view = room[1:-1].view(t.shape)
        view.copy_(t)
        return room, view

    out, mean, rstd = gpu.layernorm_train(x, **v)
    xs, vs = shifted(x)[1], {k: shifted(t)[1] for k, t in v.items()}
    room, o = shifted(torch.zeros_like(x))
    got = gpu.layernorm_train(xs, **vs, out=o)
    # sums over other lanes' shares: each off by fp32's bar of the forward test, then one rounding of the output's type
    bar = 2.0 ** -6 if dtype == BF16 else 1e-5
    assert (got[0].double() - out.double()).abs().max() <= bar * out.double().abs().max()
    assert room[0] == 3.0 and room[-1] == 3.0
    vs.pop("shift")
    a = gpu.layernorm_backward(dy, x, mean, rstd, weight=v["weight"], bias=v["bias"], scale=v["scale"])
    room, d = shifted(torch.zeros_like(x))
    b = gpu.layernorm_backward(shifted(dy)[1], xs, shifted(mean)[1], shifted(rstd)[1], **vs, dx=d)
    for k in a:
        step = 2.0 ** -6 if k == "dx" and dtype == BF16 else 1e-4
        assert (a[k].double() - b[k].double()).abs().max() <= step * a[k].double().abs().max(), k
    assert room[0] == 3.0 and room[-1] == 3.0


def test_no_rows(gpu):
    x = torch.empty((0, 300), dtype=BF16, device="cuda")
    s = torch.ones(300, dtype=BF16, device="cuda")
    out, mean, rstd = gpu.layernorm_train(x, shift=s, scale=s)
    assert out.shape == (0, 300) and mean.shape == (0,)
    g = gpu.layernorm_backward(x, x, mean, rstd, scale=s)
    assert g["dx"].shape == (0, 300) and not g["dscale"].any() and not g["dshift"].any()


@pytest.mark.parametrize("c", [1536, 1000])
def test_streams_and_graphs(gpu, c):
    x, v, dy, _ = _case(500, c, BF16, False, True, 9)
    shift = v["shift"]
    x8 = gpu.quantize_fp8(x)

    def step(x, x8, **kw):
        out, mean, rstd = gpu.layernorm_train(x, shift=shift, scale=v["scale"], **kw)
        a = gpu.layernorm_backward(dy, x, mean, rstd, scale=v["scale"], **kw)
        b = gpu.layernorm_backward(dy, x8, mean, rstd, scale=v["scale"], **kw)
        return [out, mean, rstd] + [t for d in (a, b) for t in d.values() if t is not None]

    want = step(x, x8)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    got = step(x, x8, stream=side)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    gr = torch.cuda.CUDAGraph()
    hold = x.clone()
    with torch.cuda.graph(gr):
        out = step(hold, gpu.quantize_fp8(hold))
    y = torch.randn_like(x)
    want_y = step(y, gpu.quantize_fp8(y))
    for src, res in ((y, want_y), (x, want)):
        hold.copy_(src)
        gr.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, res))


@pytest.mark.parametrize("m,c,n", [(300, 256, 384), (777, 1536, 1000)])
def test_a_training_step_of_norm_and_linear_in_8_bits(gpu, m, c, n):
    """norm -> quantise (both forms) -> linear, and back: input gradient through the transposed weight, weight gradient
    from the 8-bit checkpoint, norm gradient from the 8-bit form of the norm's input. Each stage against 64 bits from the
    values that the stage before it left, and the whole against 64-bit autograd of the same layer without any
    quantisation: the three quantised operands are off by at most 2^-4 of each value (e4m3's half step), rms under
    2^-5, and meet in sums of random sign, so the gradients' direction is kept: cosine above 1 - 2 * 2^-8 > 0.99."""
    x, v, _, g = _case(m, c, BF16, False, True, m)
    w = torch.randn((n, c), generator=g, device="cuda") / c ** 0.5
    dy = (torch.randn((m, n), generator=g, device="cuda") * 1e-3).to(BF16)
    w8, w8t = gpu.quantize_fp8_both(w, square=True)
    h, mean, rstd = gpu.layernorm_train(x, **v)
    h8, h8t = gpu.quantize_fp8_both(h)
    y = gpu.linear_fp8(h8, w8)
    x8 = gpu.quantize_fp8(x)
    dy8, dy8t = gpu.quantize_fp8_both(dy)
    dh = gpu.linear_fp8(dy8, w8t)
    dw = gpu.linear_fp8(dy8t, h8t, out_dtype=F32)
    grads = gpu.layernorm_backward(dh, x8, mean, rstd, scale=v["scale"])

    f = lambda t: gpu.dequantize_fp8(t, dtype=F32).double()  # noqa: E731
    assert torch.equal(f(w8t), f(w8).t())
    for got, a, b, k in ((y, h8, w8, c), (dh, dy8, w8t, n), (dw, dy8t, h8t, m)):
        want, size = ref.linear(f(a), f(b))
        err = (k + 8) * 2 * U * size
        _within(got, want, err, got.dtype)

    leaves = {"x": x.double(), "w": w.double(), "shift": v["shift"].double(), "scale": v["scale"].double()}
    for t in leaves.values():
        t.requires_grad_(True)
    whole = ref.norm(leaves["x"], shift=leaves["shift"], scale=leaves["scale"])[0] @ leaves["w"].t()
    whole.backward(dy.double())
    for got, want in ((dw, leaves["w"].grad), (grads["dx"], leaves["x"].grad), (grads["dscale"], leaves["scale"].grad),
                      (grads["dshift"], leaves["shift"].grad), (y, whole.detach())):
        a, b = got.double().flatten(), want.flatten()
        assert float(a @ b / (a.norm() * b.norm())) > 0.99
    gpu.device_check()


def _placed(t, off, fill):
    """t as a view that starts off elements past a 16-byte boundary, between elements of the value fill."""
    room = torch.full((t.numel() + 32,), fill, dtype=t.dtype, device="cuda")
    view = room[8 + off:8 + off + t.numel()].view(t.shape)
    view.copy_(t)
    return room, view


def _untouched(room, off, n, fill):
    return bool((room[:8 + off] == fill).all() and (room[8 + off + n:] == fill).all())


PLACES = [(0, 0, 0), (1, 1, 1), (3, 3, 3), (1, 0, 2), (0, 3, 0)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,c", [(1, 3), (2, 7), (9, 8), (10, 257), (65, 130), (130, 12), (70, 1531), (33, 4095), (3, 4096),
                                 (40, 4101), (5, 8185), (5, 8191), (3, 8192)])
def test_rows_at_any_offset_between_values_that_are_not_theirs(gpu, m, c, dtype):
    """Rows whose ends share 16-byte words with the next rows and with NaN before and behind the tensors, all tensors off
    the grid alike or each by another amount: the formulas with the bars of the tests above, and nothing written outside."""
    x, v, dy, _ = _case(m, c, dtype, True, True, 11 + m + c)
    want, mean_w, rstd_w = ref.norm(x, **v)
    xd = x.double()
    size = xd.abs().mean(1)
    n = (xd - mean_w[:, None]) * rstd_w[:, None]
    rel = (D + 8) * U + (rstd_w * D * U * size) ** 2
    e_n = rstd_w[:, None] * (D * U * size[:, None] + 2 * U * (xd - mean_w[:, None]).abs()) + rel[:, None] * n.abs()
    w, b, s1, sh = _vec(v, x)
    bar = (w * s1).abs() * e_n + 4 * U * ((n * w * s1).abs() + (b * s1).abs() + sh.abs())
    vb = {k: t for k, t in v.items() if k != "shift"}
    x8 = gpu.quantize_fp8(x)
    for at_x, at_out, at_dy in PLACES:
        xs, dys = _placed(x, at_x, float("nan"))[1], _placed(dy, at_dy, float("nan"))[1]
        room, out = _placed(torch.zeros_like(x), at_out, 3.0)
        _, mean, rstd = gpu.layernorm_train(xs, **v, out=out)
        _within(mean, mean_w, D * U * size)
        _within(rstd, rstd_w, rel * rstd_w)
        _within(out, want, bar, dtype)
        assert _untouched(room, at_out, x.numel(), 3.0)
        for inp, values in ((xs, x), (x8, gpu.dequantize_fp8(x8, dtype=F32))):
            room, dx = _placed(torch.zeros_like(x), at_out, 3.0)
            got = gpu.layernorm_backward(dys, inp, mean, rstd, **vb, dx=dx)
            assert got["dx"].data_ptr() == dx.data_ptr() and _untouched(room, at_out, x.numel(), 3.0)
            bars = _backward_bars(dy, values, mean, rstd, vb)
            for k, t in ref.norm_backward(dy, values, mean, rstd, **vb).items():
                _within(got[k], t, bars[k], dtype if k == "dx" else F32)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("m,c", [(6, 5), (20, 129), (40, 1531), (12, 4099)])
@pytest.mark.parametrize("off", [0, 1])
def test_a_row_of_nan_leaves_its_neighbours(gpu, m, c, dtype, off):
    x, v, dy, _ = _case(m, c, dtype, True, False, 12 + c)
    out, mean, rstd = gpu.layernorm_train(x, **v)
    x_bad, dy_bad = x.clone(), dy.clone()
    x_bad[m // 2], dy_bad[m // 2] = float("nan"), float("inf")
    bad = _placed(x_bad, off, 0.0)[1]
    got, mean_b, rstd_b = gpu.layernorm_train(bad, **v, out=_placed(out, off, 0.0)[1])
    rest = torch.arange(m, device="cuda") != m // 2
    assert torch.equal(mean_b[rest].isnan().any(), torch.tensor(False, device="cuda")) and mean_b[~rest].isnan().all()
    v.pop("shift"), v.pop("scale")
    dx = gpu.layernorm_backward(dy, x, mean, rstd, **v)["dx"]
    dx_b = gpu.layernorm_backward(_placed(dy_bad, off, 0.0)[1], bad, mean_b, rstd_b, **v, dx=_placed(dx, off, 0.0)[1])["dx"]
    assert got[~rest].isnan().all() and dx_b[~rest].isnan().all()
    if off == 0:  # the same rows in the same threads: the same bits
        assert torch.equal(got[rest], out[rest]) and torch.equal(dx_b[rest], dx[rest])
    assert torch.isfinite(got[rest]).all() and torch.isfinite(dx_b[rest]).all()
