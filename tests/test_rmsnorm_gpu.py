"""RMS norm (lsc_rmsnorm) against its definition in 64 bits.

Tolerances, from counting roundings (u = 2^-24): h = x + r is one rounding (u, relative to h); the
sum of squares adds d terms in at most d / 64 + 32 steps one after another on any path, so
its relative error is below (d / 64 + 32) u, halved by the square root; dividing, the root, its
reciprocal and the two products with gamma add 8 u.  Outputs in 16 bits add half a step of their
type (2^-11, 2^-8), and 2^-25 where f16 is subnormal.  An int8 code is within half a step of y / s
plus the relative error of both."""
import pytest

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
HALF_STEP = {"float32": U, "float16": 2.0 ** -11, "bfloat16": 2.0 ** -8}


def _rel(d):
    return (d / 128 + 26) * U


def _make(rows, d, xt, rt, seed, pad=0, device="cuda:0"):
    import torch
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, d + pad, generator=g).to(getattr(torch, xt)).to(device)[:, :d]
    r = None if rt is None else (2 * torch.randn(rows, d + pad, generator=g)).to(getattr(torch, rt)).to(device)[:, :d]
    gamma = (1 + 0.1 * torch.randn(d, generator=g)).to(device)
    return x, r, gamma


def _define(x, r, gamma, eps):
    h = x.double() if r is None else x.double() + r.double()
    y = h / (h.square().mean(1, keepdim=True) + eps).sqrt()
    return h, y if gamma is None else y * gamma.double()


def _close(got, want, name, rel):
    tol = want.abs() * (HALF_STEP[name] * 1.0001 + rel) + (2.0 ** -25 if name == "float16" else 0.0)
    bad = (got.double() - want).abs() > tol
    assert not bool(bad.any()), (int(bad.sum()), float(((got.double() - want).abs() - tol).max()))


def _codes(q, y, s, rel, rounding=0):
    import torch
    t = (y / s).clamp(-128, 127)
    off = (q.double() - t).abs() - 0.5 - (y / s).abs().clamp(max=128) * 2 * rel
    assert float(off.max()) <= 1e-12, float(off.max())
    clear = (t - t.floor() - 0.5).abs() > t.abs() * 2 * rel + 1e-12
    assert torch.equal(q.double()[clear], torch.floor(t[clear] + 0.5))


TYPES = [("float32", None), ("float32", "float32"), ("float16", None), ("float16", "float16"), ("float16", "float32"),
         ("bfloat16", "bfloat16"), ("bfloat16", "float32")]


@pytest.mark.parametrize("xt,rt", TYPES)
@pytest.mark.parametrize("rows,d", [(1, 1), (3, 7), (5, 64), (2, 768), (33, 1000), (1, 4096), (7, 5003), (4, 8192),
                                    (300, 264), (2, 16384), (3, 40000)])
def test_rmsnorm_types_and_sizes(cuda, rows, d, xt, rt):
    import torch
    from lightship_b200 import ops
    x, r, gamma = _make(rows, d, xt, rt, rows * 31 + d)
    h, y = _define(x, r, gamma, 1e-5)
    out = torch.empty_like(x)
    s = None if r is None else torch.empty_like(r)
    assert ops.rmsnorm(x, gamma, residual=r, sum_out=s, out=out) is out
    _close(out, y, xt, _rel(d))
    if r is not None:
        _close(s, h, rt, U)
    # the same row quantized: static scale, then its own scale
    q = torch.empty(rows, d, dtype=torch.int8, device=cuda)
    assert ops.rmsnorm(x, gamma, residual=r, out_i8=q, s_out=0.03) is q
    _codes(q, y, 0.03, _rel(d) + U)
    scales = torch.empty(rows, device=cuda)
    ops.rmsnorm(x, gamma, residual=r, out=out, out_i8=q, row_scales=scales)
    want = y.abs().amax(1) / 127
    want[want == 0] = 1.0
    assert float(((scales.double() - want).abs() / want).max()) <= _rel(d) + 2 * U
    _codes(q, y, scales.double()[:, None], _rel(d) + U)
    _close(out, y, xt, _rel(d))
    ops.check_device()


@pytest.mark.parametrize("xt,rt", [("float32", "float32"), ("float16", "float16"), ("bfloat16", "float32")])
@pytest.mark.parametrize("d,pad", [(768, 3), (768, 8), (4096, 1), (100, 4)])
def test_rmsnorm_strides_and_alignment(cuda, d, pad, xt, rt):
    """Rows apart by odd strides, and bases off the vector alignment."""
    import torch
    from lightship_b200 import ops
    x, r, gamma = _make(9, d, xt, rt, d + pad, pad)
    h, y = _define(x, r, gamma, 1e-6)
    out = torch.full((9, d + pad), 7.0, dtype=x.dtype, device=cuda)
    ops.rmsnorm(x, gamma, eps=1e-6, residual=r, out=out[:, :d])
    _close(out[:, :d], y, xt, _rel(d))
    assert bool((out[:, d:] == 7.0).all())
    x1, y1 = x[:, 1:], _define(x[:, 1:], r[:, 1:], gamma[1:].contiguous(), 1e-6)[1]
    q = torch.full((9, d + 5), 99, dtype=torch.int8, device=cuda)
    g1 = torch.empty(d, device=cuda)[1:]
    g1.copy_(gamma[1:])
    ops.rmsnorm(x1, g1, eps=1e-6, residual=r[:, 1:], out_i8=q[:, 3:d + 2], s_out=0.05)
    _codes(q[:, 3:d + 2], y1, 0.05, _rel(d) + U)
    assert bool((q[:, :3] == 99).all()) and bool((q[:, d + 2:] == 99).all())


@pytest.mark.parametrize("d", [512, 777, 4096, 40000])
@pytest.mark.parametrize("xt,rt", [("float32", "float32"), ("float16", "float16"), ("bfloat16", "float32")])
def test_rmsnorm_in_place(cuda, d, xt, rt):
    """sum_out over the residual and out over x."""
    import torch
    from lightship_b200 import ops
    x, r, gamma = _make(5, d, xt, rt, d)
    h, y = _define(x, r, gamma, 1e-5)
    ops.rmsnorm(x, gamma, residual=r, sum_out=r, out=x)
    _close(x, y, xt, _rel(d))
    _close(r, h, rt, U)


@pytest.mark.parametrize("rounding", [0, 1])
def test_rmsnorm_special_rows(cuda, rounding):
    """Rows of zeros, with NaN, with infinities, ties and codes past the int8 range."""
    import torch
    from lightship_b200 import ops
    d = 256
    x = torch.zeros(6, d, device=cuda)
    x[1] = torch.randn(d, generator=torch.Generator().manual_seed(3)).to(cuda)
    x[1, 5] = float("nan")
    x[2] = 1.0
    x[2, 9] = float("inf")
    x[3] = 1.0        # y = 1 exactly (eps = 0)
    x[4] = 2.0 ** -30
    x[5, 0] = -16.0   # the others zero: y = -16 there
    out = torch.empty_like(x)
    q = torch.empty(6, d, dtype=torch.int8, device=cuda)
    scales = torch.empty(6, device=cuda)
    ops.rmsnorm(x, eps=0.0, out=out, out_i8=q, row_scales=scales, rounding=rounding)
    o, qq, s = out.cpu(), q.cpu(), scales.cpu()
    assert bool(o[0].isnan().all()) and bool((qq[0] == 0).all()) and float(s[0]) == 1.0  # 0 / 0
    assert bool(o[1].isnan().all()) and bool((qq[1] == 0).all())
    assert bool((o[2, :9] == 0).all()) and bool(o[2, 9].isnan())
    assert bool((o[3] == 1).all()) and bool((qq[3] == 127).all()) and float(s[3]) == torch.tensor(1 / 127).item()
    assert bool((o[4] == 1).all())
    assert float(o[5, 0]) == -16.0 and int(qq[5, 0]) == -127
    # ties and saturation with a static scale: y = 1 -> 0.5 steps of 2; y = -16 -> -160
    ops.rmsnorm(x, eps=0.0, out_i8=q, s_out=2.0, rounding=rounding)
    assert bool((q[3] == (0 if rounding else 1)).all())
    ops.rmsnorm(x, eps=0.0, out_i8=q, s_out=0.1, rounding=rounding)
    assert int(q[5, 0]) == -128
    ops.rmsnorm(x, out_i8=q, row_scales=scales)  # eps > 0: a row of zeros is zeros, with scale 1
    assert bool((q[0] == 0).all()) and float(scales[0]) == 1.0
    ops.check_device()


def test_rmsnorm_many_rows_and_far_offsets(cuda):
    """More rows than one grid, and rows whose offsets pass 32 bits."""
    import torch
    from lightship_b200 import ops
    x, r, gamma = _make(70001, 40, "float16", "float16", 1)
    out = ops.rmsnorm(x, gamma, residual=r)
    _close(out, _define(x, r, gamma, 1e-5)[1], "float16", _rel(40))
    flat = torch.zeros(2 ** 32 // 2 + 4096, dtype=torch.float16, device=cuda)
    far = flat.as_strided((3, 512), (2 ** 30, 1))  # the last row starts 2^32 bytes in
    far.copy_(torch.randn(3, 512, generator=torch.Generator().manual_seed(2)).half())
    out = ops.rmsnorm(far)
    _close(out, _define(far, None, None, 1e-5)[1], "float16", _rel(512))


def test_rmsnorm_other_stream_and_graph(cuda):
    import torch
    from lightship_b200 import ops
    x, r, gamma = _make(64, 768, "float32", "float32", 4)
    q = torch.empty(64, 768, dtype=torch.int8, device=cuda)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out = ops.rmsnorm(x, gamma, residual=r)
    s.synchronize()
    _close(out, _define(x, r, gamma, 1e-5)[1], "float32", _rel(768))
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        ops.rmsnorm(x, gamma, residual=r, sum_out=r, out_i8=q, s_out=0.03)
    want = _define(x, r, gamma, 1e-5)[1]
    g.replay()
    _codes(q, want, 0.03, _rel(768) + U)
    want = _define(x, r, gamma, 1e-5)[1]  # the residual moved on
    g.replay()
    _codes(q, want, 0.03, _rel(768) + U)


def test_rmsnorm_refusals(cuda):
    import torch
    from lightship_b200 import ops
    x = torch.zeros(4, 64, device=cuda)
    with pytest.raises(ValueError):
        ops.rmsnorm(x.double())
    with pytest.raises(ValueError):
        ops.rmsnorm(x.T)
    with pytest.raises(ValueError):
        ops.rmsnorm(x, residual=x.half())
    with pytest.raises(ValueError):
        ops.rmsnorm(x, residual=x[:2])
    with pytest.raises(ValueError):
        ops.rmsnorm(x, gamma=torch.ones(63, device=cuda))
    with pytest.raises(ValueError):
        ops.rmsnorm(x.cpu())
    from lightship_b200._lib import LightShipError
    with pytest.raises(LightShipError):
        ops.rmsnorm(x, out_i8=torch.empty(4, 64, dtype=torch.int8, device=cuda))  # no scale
    with pytest.raises(LightShipError):
        ops.rmsnorm(x, sum_out=torch.empty_like(x))  # no residual
    assert ops.rmsnorm(x[:0]).shape == (0, 64)
