"""The encoder-block operators (matrix product with epilogue, root-mean-square
norm, bucketed position bias) against plain implementations in 64 bits.

Tolerances are bounds, per element, from the number formats: u is half a
spacing of the output's type relative to its value (2^-8 bf16, 2^-11 fp16,
2^-24 fp32), each fp32 addition of a sum may lose 2^-23 of it, so a sum of n
terms is off by at most n 2^-23 times the sum of the terms' magnitudes; the
activation's own error is 3e-7; what is rounded on the way (the saved sums,
dz as an operand) adds u times its magnitude times the slope it meets
(|act'| <= 1.13, |act''| <= 0.8).
"""
import pytest
import torch
import torch.nn.functional as F

from affmae_b200.kernels.bucket_bias import BucketBias, bucket_bias, bucket_count, log_edges
from affmae_b200.kernels.linear import (FusedLinear, LinearE4M3, fused_linear, linear_e4m3, linear_status,
                                        quantize_e4m3)
from affmae_b200.kernels.rms_norm import FusedRMSNorm, fused_rms_norm, rms_norm_e4m3

U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}
TINY = {torch.bfloat16: 0.0, torch.float16: 2.0 ** -24, torch.float32: 0.0}   # fp16's spacing next to zero
E = 2.0 ** -23
BF16, FP16, FP32 = torch.bfloat16, torch.float16, torch.float32
ACT = {"none": lambda v: v, "relu": F.relu, "gelu": F.gelu, "silu": F.silu}


def rnd(dev, seed, *shape, std=1.0, dtype=FP32):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dev, dtype)


def within(got, want, tol, what=""):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} beyond the bound, worst {(err / tol).max():.3g}"


def linear_ref(x, w, b, act, res, dout=None):
    """Outputs, gradients and bounds in 64 bits."""
    t, ot = x.dtype, res.dtype if res is not None else x.dtype
    M, K, N = x.shape[0], x.shape[1], w.shape[0]
    xd, wd = x.double(), w.double()
    z = xd @ wd.T
    zerr = (K + 16) * E * (xd.abs() @ wd.abs().T)
    if b is not None:
        z = z + b.double()
        zerr = zerr + E * (z.abs() + b.double().abs())
    zl = z.clone().requires_grad_(True)
    y = ACT[act](zl)
    slope = torch.autograd.grad(y.sum(), zl)[0]
    y = y.detach()
    out = y + res.double() if res is not None else y
    out_tol = U[ot] * out.abs() + TINY[ot] + 1.13 * zerr + 3e-7 * z.abs().clamp(min=1)
    if res is not None:
        out_tol = out_tol + E * out.abs()
    if dout is None:
        return out, out_tol
    d = dout.double()
    dz = d * slope
    derr = torch.zeros_like(dz) if act == "none" else d.abs() * (0.8 * (U[t] * z.abs() + TINY[t] + zerr) + 1e-6)
    if act == "relu":  # a sum within its own error of zero may fall on either side
        derr = d.abs() * 1e-6 + torch.where(z.abs() <= zerr + TINY[t], d.abs(), torch.zeros_like(d))
    op = derr + U[t] * dz.abs() + TINY[t]        # dz as the products' operand
    ad = dz.abs() + op
    dx, dw, db = dz @ wd, dz.T @ xd, dz.sum(0)
    dx_tol = op @ wd.abs() + (N + 16) * E * (ad @ wd.abs()) + U[t] * dx.abs() + TINY[t]
    dw_tol = op.T @ xd.abs() + (M + 16) * E * (ad.T @ xd.abs()) + U[t] * dw.abs() + TINY[t]
    bt = b.dtype if b is not None else t
    db_tol = derr.sum(0) + (M + 16) * E * ad.sum(0) + U[bt] * db.abs() + TINY[bt]
    return out, out_tol, dx, dx_tol, dw, dw_tol, db, db_tol


# (rows, out, in): single values, few rows, ragged tiles, several column tiles, a long sum over rows
SHAPES = [(1, 1, 1), (1, 17, 33), (3, 64, 128), (8, 96, 200), (9, 16, 16), (9, 1, 5), (127, 24, 40), (128, 256, 64),
          (129, 192, 96), (200, 100, 72), (300, 257, 65), (257, 768, 384), (70001, 32, 24), (1000, 520, 136),
          (283, 2, 1), (65, 2, 2)]   # the last: sums of two terms, where the slope's own error shows


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape", SHAPES)
@pytest.mark.parametrize("act", ["none", "gelu"])
def test_linear_forward_and_gradients(cuda, dtype, shape, act):
    M, N, K = shape
    x, w, b = rnd(cuda, 1, M, K, dtype=dtype), rnd(cuda, 2, N, K, std=K ** -0.5, dtype=dtype), rnd(cuda, 3, N, dtype=dtype)
    dout = rnd(cuda, 4, M, N, dtype=dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = fused_linear(*leaves, act=act)
    grads = torch.autograd.grad(y, leaves, dout)
    out, out_tol, dx, dx_tol, dw, dw_tol, db, db_tol = linear_ref(x, w, b, act, None, dout)
    assert y.dtype == dtype and [g.dtype for g in grads] == [dtype] * 3
    within(y, out, out_tol, "y")
    within(grads[0], dx, dx_tol, "dx")
    within(grads[1], dw, dw_tol, "dw")
    within(grads[2], db, db_tol, "db")
    assert linear_status()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("shape", [(5000, 256, 192), (20011, 640, 448), (2000, 1024, 96), (900, 1032, 64),
                                   (600, 384, 520)])
@pytest.mark.parametrize("act", ["relu", "gelu", "silu"])
def test_linear_gradients_of_larger_layers(cuda, dtype, shape, act):
    """Several tiles a block, blocks in pairs, and columns that do not fill the last tile."""
    M, N, K = shape
    x, w, b = rnd(cuda, 1, M, K, dtype=dtype), rnd(cuda, 2, N, K, std=K ** -0.5, dtype=dtype), rnd(cuda, 3, N, dtype=dtype)
    dout = rnd(cuda, 4, M, N, dtype=dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = fused_linear(*leaves, act=act)
    grads = torch.autograd.grad(y, leaves, dout)
    out, out_tol, dx, dx_tol, dw, dw_tol, db, db_tol = linear_ref(x, w, b, act, None, dout)
    within(y, out, out_tol, "y")
    within(grads[0], dx, dx_tol, "dx")
    within(grads[1], dw, dw_tol, "dw")
    within(grads[2], db, db_tol, "db")
    again = torch.autograd.grad(fused_linear(*leaves, act=act), leaves, dout)
    assert all(torch.equal(p, q) for p, q in zip(grads, again))
    assert linear_status()


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(4, 48, 32), (131, 200, 64), (140, 77, 33)])
@pytest.mark.parametrize("act", ["none", "relu", "gelu", "silu"])
@pytest.mark.parametrize("types", [(BF16, BF16, BF16), (BF16, FP32, FP32), (FP16, FP32, FP16), (FP32, FP32, FP32),
                                   (FP16, None, FP32)])
def test_linear_residual_bias_and_output_types(cuda, shape, act, types):
    dtype, bias_dtype, res_dtype = types
    M, N, K = shape
    x, w = rnd(cuda, 5, M, K, dtype=dtype), rnd(cuda, 6, N, K, std=K ** -0.5, dtype=dtype)
    b = rnd(cuda, 7, N, dtype=bias_dtype) if bias_dtype else None
    res = rnd(cuda, 8, M, N, dtype=res_dtype)
    dout = rnd(cuda, 9, M, N, dtype=res_dtype)
    leaves = [t.clone().requires_grad_(True) if t is not None else None for t in (x, w, b, res)]
    y = fused_linear(leaves[0], leaves[1], leaves[2], act, leaves[3])
    assert y.dtype == res_dtype
    grads = torch.autograd.grad(y, [t for t in leaves if t is not None], dout)
    out, out_tol, dx, dx_tol, dw, dw_tol, db, db_tol = linear_ref(x, w, b, act, res, dout)
    within(y, out, out_tol, "y")
    within(grads[0], dx, dx_tol, "dx")
    within(grads[1], dw, dw_tol, "dw")
    if b is not None:
        within(grads[2], db, db_tol, "db")
    assert torch.equal(grads[-1], dout)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("rows", [5, 200])
def test_linear_strided_unaligned_and_batched_inputs(cuda, dtype, rows):
    K, N = 48, 40
    base = rnd(cuda, 10, rows, 2 * K, dtype=dtype)
    wide = rnd(cuda, 11, K, N, dtype=dtype) * K ** -0.5
    flat = rnd(cuda, 12, rows * N + 1, dtype=dtype)
    xs, wt, res = base[:, ::2], wide.t(), flat[1:].view(rows, N)   # strided, transposed, off by one element
    off = torch.empty(rows * K + 3, device=cuda, dtype=dtype)[3:].view(rows, K).copy_(xs)
    out, tol = linear_ref(xs.contiguous(), wt.contiguous(), None, "silu", res)
    for x in (xs, off):
        within(fused_linear(x, wt, None, "silu", res), out, tol)
        y = fused_linear(x.reshape(1, rows, K), wt, None, "silu", res.reshape(1, rows, N))
        within(y[0], out, tol)
    d = torch.randn(1, device=cuda).to(dtype).expand(rows, N)       # a broadcast gradient
    x = xs.detach().clone().requires_grad_(True)
    (g,) = torch.autograd.grad(fused_linear(x, wt, None), (x,), d)
    ref = linear_ref(x.detach(), wt.contiguous(), None, "none", None, d.contiguous())
    within(g, ref[2], ref[3])


@pytest.mark.gpu
def test_linear_partial_gradients_and_empty_rows(cuda):
    x, w, b = rnd(cuda, 13, 130, 64, dtype=BF16), rnd(cuda, 14, 32, 64, dtype=BF16), rnd(cuda, 15, 32, dtype=BF16)
    dout = rnd(cuda, 16, 130, 32, dtype=BF16)
    full = [t.clone().requires_grad_(True) for t in (x, w, b)]
    want = torch.autograd.grad(fused_linear(*full, act="gelu"), full, dout)
    for i in range(3):
        part = [t.clone().requires_grad_(i == j) for j, t in enumerate((x, w, b))]
        (got,) = torch.autograd.grad(fused_linear(*part, act="gelu"), [part[i]], dout)
        assert torch.equal(got, want[i])
    empty = torch.empty((0, 64), device=cuda, dtype=BF16, requires_grad=True)
    full = [empty] + [t.clone().requires_grad_(True) for t in (w, b)]
    y = fused_linear(*full, act="gelu")
    assert y.shape == (0, 32)
    dx, dw, db = torch.autograd.grad(y, full, y.detach())
    assert dx.shape == (0, 64) and not dw.any() and not db.any()


@pytest.mark.gpu
def test_linear_nonfinite_rows_stay_in_their_rows(cuda):
    x, w = rnd(cuda, 17, 150, 96, dtype=BF16), rnd(cuda, 18, 64, 96, dtype=BF16)
    clean = {a: fused_linear(x, w, None, a) for a in ACT}
    x[3, 5], x[140, 0] = float("nan"), float("inf")
    keep = torch.ones(150, dtype=torch.bool, device=cuda)
    keep[[3, 140]] = False
    for a in ACT:
        y = fused_linear(x, w, None, a)
        assert torch.equal(y[keep], clean[a][keep]) and y[3].isnan().all()
    assert torch.equal(fused_linear(x, w)[140], torch.where(w[:, 0] > 0, float("inf"), float("-inf")).to(BF16))


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_linear_gradients_of_huge_sums(cuda, act):
    """Sums beyond fp16's range (in which bf16 layers keep them): the slope is 1 above and 0 below."""
    x = torch.full((64, 32), 300.0, device=cuda, dtype=BF16).requires_grad_(True)
    w = torch.full((16, 32), 50.0, device=cuda, dtype=BF16)
    w[::2] *= -1
    dout = rnd(cuda, 35, 64, 16, dtype=BF16)
    y = fused_linear(x, w, None, act)
    (dx,) = torch.autograd.grad(y, x, dout)
    assert (y[:, 1::2] == torch.tensor(32 * 300 * 50.0, device=cuda).to(BF16)).all() and not y[:, ::2].any()
    want = dout.double()[:, 1::2].sum(1, keepdim=True) * 50
    within(dx, want.expand(-1, 32), 8 * E * 50 * dout.double().abs().sum(1, keepdim=True) + U[BF16] * want.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("act", ["gelu", "silu"])
def test_linear_gradients_against_differences(cuda, act):
    """Directional differences of the fp32 forward: the central difference's own error is h^2 / 6 of the third
    derivative along the direction (of order one, h = 2^-6: 4e-5) and 2^-22 / h of the sum's magnitude."""
    M, N, K = 150, 40, 24
    x, w, b = rnd(cuda, 19, M, K), rnd(cuda, 20, N, K, std=K ** -0.5), rnd(cuda, 21, N)
    dout = rnd(cuda, 22, M, N)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    grads = torch.autograd.grad(fused_linear(*leaves, act=act), leaves, dout)
    h = 2.0 ** -6
    for i, t in enumerate((x, w, b)):
        v = rnd(cuda, 23 + i, *t.shape)
        v = v / (1 if i == 2 else K ** 0.5 if i == 0 else 1)

        def f(s):
            a = [x, w, b]
            a[i] = t + s * h * v
            return (fused_linear(*a, act=act).double() * dout.double())
        terms = (f(1) - f(-1)) / (2 * h)
        want = (grads[i].double() * v.double()).sum()
        # the truncation errors of the M N terms have no common sign: sqrt of their number, times 8
        scale = dout.double().norm() * max(1.0, float(v.double().norm() / v[..., 0].numel() ** 0.5) ** 3)
        assert abs(terms.sum() - want) <= 8 * scale * (h * h / 6 * 8 + E / h * 4)


@pytest.mark.gpu
def test_linear_on_a_side_stream_and_repeatable(cuda):
    x, w, b = rnd(cuda, 27, 4096, 96, dtype=BF16), rnd(cuda, 28, 64, 96, dtype=BF16), rnd(cuda, 29, 64, dtype=BF16)
    dout = rnd(cuda, 30, 4096, 64, dtype=BF16)

    def step():
        leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
        y = fused_linear(*leaves, act="gelu")
        return [y, *torch.autograd.grad(y, leaves, dout)]
    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    for a, b_ in zip(got, want):
        assert torch.equal(a, b_)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", [(4000, 256, 96), (20000, 512, 64), (40000, 1024, 24), (100, 40000, 8), (120, 20000, 72)])
def test_linear_wide_tiles_with_saved_sums_or_residual(cuda, dtype, shape):
    """Tiles as wide as they get beside two staging buffers a warp, by single blocks and by pairs."""
    M, N, K = shape
    x, w, b = rnd(cuda, 1, M, K, dtype=dtype), rnd(cuda, 2, N, K, std=K ** -0.5, dtype=dtype), rnd(cuda, 3, N, dtype=dtype)
    res = rnd(cuda, 4, M, N)
    y = fused_linear(x.clone().requires_grad_(True), w, b, "gelu").detach()
    z = fused_linear(x, w, b, "silu", res)
    out, tol = linear_ref(x, w, b, "gelu", None)
    within(y, out, tol, "gelu")
    out, tol = linear_ref(x, w, b, "silu", res)
    within(z, out, tol, "residual")
    assert linear_status()


@pytest.mark.gpu
def test_linear_as_a_threads_first_call(cuda):
    """A thread that has made no CUDA call of its own yet (as autograd's have not) may begin with a product."""
    import threading
    x, w = rnd(cuda, 33, 256, 64, dtype=BF16), rnd(cuda, 34, 64, 64, dtype=BF16)
    with torch.no_grad():
        want = fused_linear(x, w)
        got = []
        t = threading.Thread(target=lambda: got.append(fused_linear(x, w)))
        t.start()
        t.join()
    assert got and torch.equal(got[0], want)


@pytest.mark.gpu
def test_linear_module_follows_autocast(cuda):
    torch.manual_seed(0)
    lin = FusedLinear(96, 64, act="gelu").to(cuda)
    x, res = rnd(cuda, 31, 200, 96), rnd(cuda, 32, 200, 64)
    out, tol = linear_ref(x, lin.weight.detach(), lin.bias.detach(), "gelu", None)
    within(lin(x), out, tol)
    with torch.autocast("cuda", dtype=BF16):
        y = lin(x)
        assert y.dtype == BF16
        z = lin(x, res)
        assert z.dtype == FP32
    out, tol = linear_ref(x.to(BF16), lin.weight.detach().to(BF16), lin.bias.detach(), "gelu", res)
    within(z, out, tol)
    z.sum().backward()
    assert lin.weight.grad.dtype == FP32 and lin.bias.grad.shape == (64,)


# --------------------------------------------------------------- e4m3 -----

def e4m3_round(v):
    """Nearest e4m3 value in 64 bits (ties to even)."""
    _, e = torch.frexp(v)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return (torch.round(v / step) * step).clamp(-448, 448)


def check_e4m3(q, scale, y, yerr):
    """q, scale against the 64-bit rows y known to within yerr: the scale to its rounding, and each value one
    that some input within the error rounds to."""
    top = y.abs().amax(-1)
    want = torch.where(top > 0, top / 448, torch.ones_like(top))
    rel = (yerr.amax(-1) / top.clamp(min=1e-300)).clamp(max=1.0) + 4 * E
    assert ((scale.double() - want).abs() <= rel * want).all()
    v = y / want[..., None]
    dv = v.abs() * 2 * rel[..., None] + yerr / want[..., None]
    lo, hi = e4m3_round(v - dv), e4m3_round(v + dv)
    assert ((q.double() >= lo) & (q.double() <= hi)).all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape", [(1, 1), (3, 7), (5, 512), (300, 96), (17, 1025), (2, 9000), (4, 8200)])
def test_quantize_e4m3(cuda, dtype, shape):
    x = rnd(cuda, 40, *shape, std=3.0, dtype=dtype)
    x[0] = 0
    q, scale = quantize_e4m3(x)
    assert scale[0] == 1 and not q[0].double().any()
    check_e4m3(q, scale, x.double(), torch.zeros_like(x.double()))


@pytest.mark.gpu
@pytest.mark.parametrize("shape", [(1, 8, 16), (1, 33, 100), (7, 64, 4096), (9, 16, 16), (130, 256, 128), (200, 96, 80),
                                   (300, 300, 200), (257, 45, 33)])
@pytest.mark.parametrize("act,out_dtype,res_dtype", [("none", BF16, None), ("gelu", FP16, FP16), ("silu", FP32, BF16),
                                                     ("relu", BF16, FP32)])
def test_linear_e4m3(cuda, shape, act, out_dtype, res_dtype):
    M, N, K = shape
    q, s = quantize_e4m3(rnd(cuda, 41, M, K))
    wq, ws = quantize_e4m3(rnd(cuda, 42, N, K, std=K ** -0.5))
    b = rnd(cuda, 43, N)
    res = rnd(cuda, 44, M, N, dtype=res_dtype) if res_dtype else None
    y = linear_e4m3(q, s, wq, ws, b, act, res, out_dtype)
    x, w = q.double() * s.double()[:, None], wq.double() * ws.double()[:, None]
    z = x @ w.T + b.double()
    zerr = (K + 16) * E * (x.abs() @ w.abs().T) + 4 * E * (z.abs() + b.double().abs())
    out = ACT[act](z) + (res.double() if res is not None else 0)
    tol = (U[out_dtype] + E) * out.abs() + TINY[out_dtype] + 1.13 * zerr + 3e-7 * z.abs().clamp(min=1)
    assert y.dtype == out_dtype
    within(y, out, tol)
    assert linear_status()


@pytest.mark.gpu
def test_linear_e4m3_module(cuda):
    torch.manual_seed(1)
    lin = FusedLinear(256, 96, act="gelu").to(cuda)
    norm = FusedRMSNorm(256).to(cuda)
    x = rnd(cuda, 45, 2, 50, 256)
    q, s = norm.quantized(x)
    y = LinearE4M3.from_linear(lin)(q, s)
    ref = lin(norm(x))
    # two e4m3 operands (relative error 2^-4 each) average out over 256 terms
    assert y.shape == (2, 50, 96) and y.dtype == BF16
    assert (y.double() - ref.double()).norm() < 2 * 2.0 ** -4 * ref.double().norm()


# --------------------------------------------------------------- norm -----

def norm_ref(x, w, eps, delta, f, dy=None, ds=None):
    """s, y and gradients with bounds, 64 bits.  yerr is y's error before its rounding."""
    C = x.shape[-1]
    leaves = [t.double().requires_grad_(True) for t in (x, w)]
    d = delta.double().requires_grad_(True) if delta is not None else None
    fr = f.double().repeat_interleave(x.shape[0] // f.numel())[:, None] if f is not None else 1.0
    s = leaves[0] + fr * d if d is not None else leaves[0]
    r = torch.rsqrt(s.square().mean(-1, keepdim=True) + eps)
    y = s * r * leaves[1]
    sd, yd, rd = s.detach(), y.detach(), r.detach()
    serr = 2 * E * (x.double().abs() + (fr * d.detach()).abs()) if d is not None else torch.zeros_like(sd)
    # the sum of squares of C positive terms, its root and the products
    rel = (C + 16) * E
    yerr = yd.abs() * rel + serr * rd * w.double().abs() + yd.abs() * (serr * sd.abs()).mean(-1, keepdim=True) * rd ** 2
    if dy is None:
        return sd, serr, yd, yerr
    grads = torch.autograd.grad((s, y) if ds is not None else y, leaves + ([d] if d is not None else []),
                                (ds.double(), dy.double()) if ds is not None else dy.double())
    # the sum is that of the forward, unrounded: relative error u of s, once in each factor s and r of the formula
    u = rel
    g = dy.double() * w.double()
    gs = (g * sd).abs().mean(-1, keepdim=True)
    dx_err = rd * (g.abs() * 2 * rel + 4 * u * sd.abs() * rd ** 2 * gs) + rel * grads[0].abs() + \
        (2 * E * ds.double().abs() if ds is not None else 0)
    dw_err = ((dy.double() * sd * rd).abs() * (u + 4 * E)).sum(0) + (x.shape[0] + 16) * E * (dy.double() * sd * rd).abs().sum(0)
    return sd, serr, yd, yerr, grads, dx_err, dw_err


@pytest.mark.gpu
@pytest.mark.parametrize("types", [(FP32, BF16, BF16), (BF16, BF16, BF16), (FP16, FP16, FP16), (FP32, FP32, FP32),
                                   (BF16, None, FP32), (FP32, None, BF16), (BF16, FP32, FP16)])
@pytest.mark.parametrize("shape", [(1, 1), (2, 5), (4, 96), (1030, 96), (6, 384), (3, 1000), (4, 1025), (3, 4096),
                                   (2, 8192), (2, 9000), (4, 8193)])
def test_rms_norm_forward_and_gradients(cuda, types, shape):
    xt, dt, yt = types
    R, C = shape
    x, w = rnd(cuda, 50, R, C, std=2.0, dtype=xt), 1 + rnd(cuda, 51, C, std=0.2)
    delta = rnd(cuda, 52, R, C, dtype=dt) if dt else None
    f = torch.tensor([0.0, 1.25], device=cuda) if dt and R % 2 == 0 else None
    dy = rnd(cuda, 53, R, C, dtype=yt)
    ds = rnd(cuda, 54, R, C, dtype=xt) if dt else None
    leaves = [t.clone().requires_grad_(True) for t in (x, w)] + ([delta.clone().requires_grad_(True)] if dt else [])
    got = fused_rms_norm(leaves[0], leaves[1], 1e-6, leaves[2] if dt else None, f, yt)
    s, y = got if dt else (None, got)
    grads = torch.autograd.grad(got, leaves, (ds, dy) if dt else dy)
    sd, serr, yd, yerr, want, dx_err, dw_err = norm_ref(x, w, 1e-6, delta, f, dy, ds)
    if dt:
        assert s.dtype == xt
        within(s, sd, serr + U[xt] * sd.abs() + TINY[xt], "s")
    assert y.dtype == yt
    within(y, yd, yerr + U[yt] * yd.abs() + TINY[yt], "y")
    within(grads[0], want[0], dx_err + U[xt] * want[0].abs() + TINY[xt], "dx")
    within(grads[1], want[1], dw_err + U[FP32] * want[1].abs(), "dw")
    if dt:
        fr = f.double().repeat_interleave(R // 2)[:, None] if f is not None else 1.0
        within(grads[2], want[2], fr * dx_err + (U[dt] + E) * want[2].abs() + TINY[dt], "ddelta")


@pytest.mark.gpu
def test_rms_norm_single_gradients_match(cuda):
    x, w, d = rnd(cuda, 55, 64, 96), 1 + rnd(cuda, 56, 96, std=0.1), rnd(cuda, 57, 64, 96, dtype=BF16)
    dy, ds = rnd(cuda, 58, 64, 96), rnd(cuda, 59, 64, 96)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, d)]
    s, y = fused_rms_norm(leaves[0], leaves[1], delta=leaves[2])
    only_y = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    only_s = torch.autograd.grad(s, leaves, ds, retain_graph=True)
    both = torch.autograd.grad((s, y), leaves, (ds, dy))
    assert torch.equal(only_s[0], ds) and not only_s[1].any()
    assert torch.allclose(only_y[0] + only_s[0], both[0], rtol=0, atol=1e-5)
    assert torch.equal(only_y[1], both[1])


@pytest.mark.gpu
def test_rms_norm_zero_nan_and_empty_rows(cuda):
    x = rnd(cuda, 60, 5, 96)
    x[0], x[1, 7], x[2, 3] = 0, float("nan"), float("inf")
    w = torch.ones(96, device=cuda)
    y = fused_rms_norm(x, w)
    assert not y[0].any() and y[1].isnan().all() and y[2, 3].isnan() and not y[2, :3].any()
    q, scale = rms_norm_e4m3(x, w)
    assert scale[0] == 1 and not q[0].float().any() and scale[1].isnan() and q[1].float().isnan().all()
    assert torch.equal(fused_rms_norm(x[3:], w), y[3:])
    assert fused_rms_norm(x[:0], w).shape == (0, 96)
    e = torch.empty((0, 96), device=cuda, requires_grad=True)
    wl = w.clone().requires_grad_(True)
    gx, gw = torch.autograd.grad(fused_rms_norm(e, wl), (e, wl), torch.empty((0, 96), device=cuda))
    assert gx.shape == (0, 96) and not gw.any()


@pytest.mark.gpu
@pytest.mark.parametrize("types", [(BF16, BF16), (FP32, BF16), (FP16, None)])
@pytest.mark.parametrize("shape", [(1, 512), (3, 33), (200, 96), (5, 4096), (2, 8200)])
def test_rms_norm_e4m3(cuda, types, shape):
    xt, dt = types
    x, w = rnd(cuda, 61, *shape, dtype=xt), 1 + rnd(cuda, 62, shape[1], std=0.2)
    delta = rnd(cuda, 63, *shape, dtype=dt) if dt else None
    got = rms_norm_e4m3(x, w, 1e-6, delta)
    sd, serr, yd, yerr = norm_ref(x, w, 1e-6, delta, None)
    if dt:
        within(got[0], sd, serr + U[xt] * sd.abs() + TINY[xt])
    check_e4m3(got[-2], got[-1], yd, yerr)


@pytest.mark.gpu
def test_rms_norm_gradient_against_differences(cuda):
    """Central differences of the 64-bit sum of the fp32 forward, h = 2^-7 (see the linear's test)."""
    R, C = 40, 96
    x, w, d = rnd(cuda, 64, R, C), 1 + rnd(cuda, 65, C, std=0.1), rnd(cuda, 66, R, C)
    dy, ds = rnd(cuda, 67, R, C), rnd(cuda, 68, R, C)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, d)]
    grads = torch.autograd.grad(fused_rms_norm(leaves[0], leaves[1], delta=leaves[2]), leaves, (ds, dy))
    h = 2.0 ** -7
    for i in range(3):
        v = rnd(cuda, 69 + i, *leaves[i].shape)

        def f(sign):
            a = [x, w, d]
            a[i] = a[i] + sign * h * v
            s, y = fused_rms_norm(a[0], a[1], delta=a[2])
            return (s.double() * ds.double()).sum() + (y.double() * dy.double()).sum()
        want = (grads[i].double() * v.double()).sum()
        scale = dy.double().norm() + ds.double().norm()
        assert abs((f(1) - f(-1)) / (2 * h) - want) <= 8 * scale * (h * h / 6 * 8 + E / h * 4)


# --------------------------------------------------------------- bias -----

def rows_ref(edges, qp, kp, member, one):
    """Table rows [B,Nq,M] by counting edges one by one, -1 where the index is out of range."""
    B, Nq, A = qp.shape
    Nk = kp.shape[1]
    if member is None:
        pair = kp[:, None].expand(B, Nq, Nk, A)
        ok = torch.ones((B, Nq, Nk), dtype=torch.bool, device=qp.device)
    else:
        ok = (member >= 0) & (member < Nk)
        idx = torch.where(ok, member.long(), 0).view(B, -1, 1).expand(-1, -1, A)
        pair = kp.gather(1, idx).view(*member.shape, A)
    n = bucket_count(edges, 1, one)
    row = 0
    for a in reversed(range(A)):
        d = pair[..., a] - qp[:, :, None, a]
        d = torch.round(d).long() if d.is_floating_point() else d
        dist = (-d).clamp(min=0) if one else d.abs()
        c = sum((dist >= e).long() for e in edges)
        row = row * n + (c if one else len(edges) + d.sign() * c)
    return torch.where(ok, row, -1)


BIAS_CASES = [  # B, H, Nq, Nk, M (0: all keys), axes, edges, one sided, position type
    (2, 3, 50, 50, 48, 2, log_edges(7, 24), False, FP32),
    (1, 1, 1, 1, 0, 1, (1,), False, torch.int64),
    (2, 5, 1, 1000, 0, 1, log_edges(31, 4096), True, torch.int64),
    (2, 16, 37, 129, 0, 1, log_edges(15, 128), False, torch.int32),
    (1, 6, 300, 40, 5, 2, (1, 2, 5), False, FP32),
    (1, 4, 64, 64, 64, 2, log_edges(32, 60), False, FP32),       # 65 x 65 rows
    (3, 2, 9, 77, 0, 1, (3, 20000, 1 << 30), False, torch.int64),  # edges beyond the byte table
    (2, 12, 200, 200, 8, 2, (1, 4), True, torch.int32),
]


def bias_inputs(dev, case, seed=80):
    B, H, Nq, Nk, M, A, edges, one, pt = case
    g = torch.Generator().manual_seed(seed)
    span = 40 if A == 2 else 4 * Nk
    base = (1 << 41) if pt == torch.int64 else 0
    qp = (torch.randint(0, span, (B, Nq, A), generator=g) + base).to(dev, pt)
    kp = (torch.randint(0, span, (B, Nk, A), generator=g) + base).to(dev, pt)
    if len(edges) == 3 and edges[1] == 20000:
        kp[:, ::3] += 30000
        kp[:, 1::9] -= 1 << 40
    member = torch.randint(-2, Nk + 2, (B, Nq, M), generator=g).to(dev, torch.int32) if M else None
    return qp, kp, member


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("case", BIAS_CASES)
def test_bucket_bias_and_table_gradient(cuda, dtype, case):
    B, H, Nq, Nk, M, A, edges, one, _ = case
    qp, kp, member = bias_inputs(cuda, case)
    rows = bucket_count(edges, A, one)
    table = rnd(cuda, 81, rows, H, dtype=dtype).requires_grad_(True)
    bias = bucket_bias(table, edges, qp, kp, member, one)
    row = rows_ref(edges, qp, kp, member, one)
    want = torch.where((row >= 0)[..., None], table.detach()[row.clamp(min=0)], 0).permute(0, 3, 1, 2)
    assert bias.dtype == dtype and torch.equal(bias, want)
    dout = rnd(cuda, 82, *bias.shape, dtype=dtype)
    (dt,) = torch.autograd.grad(bias, (table,), dout, retain_graph=True)
    (again,) = torch.autograd.grad(bias, (table,), dout)
    assert torch.equal(dt, again)
    ok = (row >= 0).reshape(-1)
    gd = dout.double().permute(0, 2, 3, 1).reshape(-1, H)[ok]
    ref = torch.zeros((rows, H), dtype=torch.float64, device=cuda).index_add_(0, row.reshape(-1)[ok], gd)
    mag = torch.zeros_like(ref).index_add_(0, row.reshape(-1)[ok], gd.abs())
    cnt = torch.zeros_like(ref).index_add_(0, row.reshape(-1)[ok], torch.ones_like(gd))
    # a term keeps 19 bits of the tile's largest (at most the overall largest); then fp32 sums
    tol = cnt * dout.double().abs().max() * 2.0 ** -19 + cnt * E * mag + U[dtype] * ref.abs() + TINY[dtype]
    within(dt, ref, tol)


@pytest.mark.gpu
def test_bucket_bias_output_type_and_empty(cuda):
    case = BIAS_CASES[0]
    qp, kp, member = bias_inputs(cuda, case)
    mod = BucketBias(3, case[6]).to(cuda)
    with torch.no_grad():
        mod.table.copy_(rnd(cuda, 83, *mod.table.shape))
    b16 = mod(qp, kp, member.long(), BF16)
    assert b16.dtype == BF16 and torch.equal(b16, mod(qp, kp, member).to(BF16))
    b16.float().sum().backward()
    assert mod.table.grad.shape == mod.table.shape
    count = (rows_ref(case[6], qp, kp, member, False) >= 0).sum()
    assert (mod.table.grad.sum(0) - count).abs().max() < 1e-3
    for q, k, m in ((qp[:, :0], kp, member[:, :0]), (qp, kp[:, :0], None), (qp[:0], kp[:0], member[:0])):
        mod.table.grad = None
        out = mod(q, k, m)
        assert out.numel() == 0
        out.sum().backward()
        assert not mod.table.grad.any()


@pytest.mark.gpu
def test_bucket_bias_nonfinite_and_small_gradients(cuda):
    """A NaN or infinity reaches its own bucket and no other; subnormal gradients are not lost to the scaling."""
    case = BIAS_CASES[0]
    qp, kp, member = bias_inputs(cuda, case)
    member = member.clamp(0, 49)
    table = torch.zeros((225, 3), device=cuda, requires_grad=True)
    bias = bucket_bias(table, case[6], qp, kp, member)
    dout = rnd(cuda, 84, *bias.shape)
    (clean,) = torch.autograd.grad(bias, (table,), dout, retain_graph=True)
    row = rows_ref(case[6], qp, kp, member, False)
    dout[0, 1, 3, 7], dout[1, 2, 5, 9] = float("nan"), float("inf")
    (dt,) = torch.autograd.grad(bias, (table,), dout, retain_graph=True)
    assert dt[row[0, 3, 7], 1].isnan() and dt[row[1, 5, 9], 2] == float("inf")
    dt[row[0, 3, 7], 1] = clean[row[0, 3, 7], 1]
    dt[row[1, 5, 9], 2] = clean[row[1, 5, 9], 2]
    assert torch.allclose(dt, clean, rtol=0, atol=1e-3)
    (small,) = torch.autograd.grad(bias, (table,), torch.full_like(dout, 1e-38))
    cnt = torch.bincount(row.reshape(-1), minlength=225)
    assert torch.allclose(small.double(), 1e-38 * cnt[:, None].double().expand(-1, 3), rtol=1e-4, atol=0)


@pytest.mark.gpu
def test_bucket_bias_gradient_against_differences(cuda):
    """The bias is linear in the table: a difference of any size is exact up to rounding."""
    case = BIAS_CASES[3]
    qp, kp, member = bias_inputs(cuda, case)
    t0, v = rnd(cuda, 85, 31, 16), rnd(cuda, 86, 31, 16)
    table = t0.clone().requires_grad_(True)
    bias = bucket_bias(table, case[6], qp, kp, member)
    dout = rnd(cuda, 87, *bias.shape)
    (dt,) = torch.autograd.grad(bias, (table,), dout)
    f = [(bucket_bias(t0 + s * v, case[6], qp, kp, member).double() * dout.double()).sum() for s in (0.5, -0.5)]
    mag = (dout.double().abs().sum() * 4)
    assert abs((f[0] - f[1]) - (dt.double() * v.double()).sum()) <= mag * 2.0 ** -19


def test_log_edges():
    assert log_edges(1, 1) == (1,) and log_edges(7, 24)[:4] == (1, 2, 3, 4) and log_edges(7, 24)[-1] == 24
    for k in (1, 2, 9, 64):
        for reach in (1, 5, 128, 8192):
            e = log_edges(k, reach)
            assert len(e) == k and all(a < b for a, b in zip((0,) + e, e))
    assert bucket_count((1, 2, 4), 2) == 49 and bucket_count((1, 2, 4), 1, True) == 4


# ----------------------------------------------------------- refusals -----

def test_refusals_on_the_host():
    x, w = torch.zeros(4, 8), torch.zeros(3, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        fused_linear(x, w)
    with pytest.raises(RuntimeError, match="activation"):
        fused_linear(x, w, act="tanh")
    with pytest.raises(RuntimeError, match="CUDA"):
        fused_rms_norm(x, torch.ones(8))
    with pytest.raises(RuntimeError, match="edges"):
        bucket_bias(torch.zeros(5, 1), (2, 2), torch.zeros(1, 1, 1), torch.zeros(1, 1, 1))
    with pytest.raises(RuntimeError, match="CUDA"):
        quantize_e4m3(x)


def test_c_entries_refuse_before_any_launch():
    from affmae_b200 import _native as nat
    with pytest.raises(RuntimeError, match="at least one"):
        nat.call("affb_linear_fwd", None, None, None, 0, None, 0, 0, 0, 4, 0, 8, None, 0, None, None, 0, None)
    with pytest.raises(RuntimeError, match="activation"):
        nat.call("affb_linear_fwd", None, None, None, 0, None, 0, 9, 0, 4, 4, 8, None, 0, None, None, 0, None)
    with pytest.raises(RuntimeError, match="operands' type or fp32"):
        nat.call("affb_linear_fwd", None, None, None, 0, None, 0, 0, 1, 4, 4, 8, None, 2, None, None, 0, None)
    with pytest.raises(RuntimeError, match="null pointer"):
        nat.call("affb_linear_bwd", None, 0, None, None, None, 0, 0, 4, 4, 8, None, None, None, 0, None, 0, None)
    with pytest.raises(RuntimeError, match="exactly one"):
        nat.call("affb_rms_norm_fwd", None, 0, None, 0, None, 0, None, 1e-6, 4, 8, None, None, None, 0, None, None, None)
    with pytest.raises(RuntimeError, match="edges"):
        nat.call("affb_bucket_bias_fwd", None, 0, None, 0, 0, None, None, 0, 1, None, 1, 1, 1, 1, 1, None, 0, None)


@pytest.mark.gpu
def test_refusals_of_shapes_and_types(cuda):
    x, w = rnd(cuda, 90, 4, 8), rnd(cuda, 91, 3, 8)
    for bad in (lambda: fused_linear(x, rnd(cuda, 92, 3, 9)), lambda: fused_linear(x, w, torch.zeros(4, device=cuda)),
                lambda: fused_linear(x.half(), w), lambda: fused_linear(x, w, residual=torch.zeros(4, 4, device=cuda)),
                lambda: fused_linear(x.bfloat16(), w.bfloat16(), residual=torch.zeros(4, 3, device=cuda).half()),
                lambda: fused_linear(x.double(), w.double()), lambda: fused_linear(x[:, :0], w[:, :0]),
                lambda: fused_rms_norm(x, torch.ones(7, device=cuda)), lambda: fused_rms_norm(x.double(), torch.ones(8, device=cuda)),
                lambda: fused_rms_norm(x, torch.ones(8, device=cuda), row_scale=torch.ones(2, device=cuda)),
                lambda: fused_rms_norm(x, torch.ones(8, device=cuda), delta=x, row_scale=torch.ones(3, device=cuda)),
                lambda: fused_rms_norm(x, torch.ones(8, device=cuda), delta=x[:2]),
                lambda: linear_e4m3(x, x[:, 0], w, w[:, 0]),
                lambda: bucket_bias(torch.zeros(4, 2, device=cuda), (1, 2), torch.zeros(1, 3, 1, device=cuda), torch.zeros(1, 3, 1, device=cuda)),
                lambda: bucket_bias(torch.zeros(5, 2, device=cuda), (1, 2), torch.zeros(1, 3, 3, device=cuda), torch.zeros(1, 3, 3, device=cuda)),
                lambda: bucket_bias(torch.zeros(5, 2, device=cuda), (1, 2), torch.zeros(1, 3, 1, device=cuda), torch.zeros(1, 3, 1, device=cuda).long())):
        with pytest.raises(RuntimeError):
            bad()
    q, s = quantize_e4m3(x)
    wq, ws = quantize_e4m3(w)
    with pytest.raises(RuntimeError):
        linear_e4m3(q, s[:2], wq, ws)
    xg = x.clone().requires_grad_(True)
    (g,) = torch.autograd.grad(fused_linear(xg, w, act="gelu").sum(), xg, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


@pytest.mark.gpu
def test_bucket_bias_nan_positions_and_no_keys(cuda):
    """A NaN position counts as the farthest key before the query, by either way of finding buckets; lists without
    any key give a bias of zero and no gradient."""
    edges = (1, 2, 5)
    pos = torch.arange(16, device=cuda).float().view(1, 16, 1).clone()
    kp = pos.clone()
    kp[0, 3] = float("nan")
    for one in (False, True):
        rows = bucket_count(edges, 1, one)
        table = rnd(cuda, 95, rows, 2)
        far = rows - 1 if one else 0
        small = bucket_bias(table, edges, pos, kp, None, one)                       # few pairs: buckets looked up
        many = bucket_bias(table, edges, pos.expand(64, -1, -1), kp.expand(64, -1, -1), None, one)  # by offset
        assert torch.equal(small[0, :, 5, 3], table[far]) and torch.equal(many[9], small[0])
    member = torch.randint(-1, 3, (1, 16, 8), device=cuda)
    table = rnd(cuda, 96, 7, 2).requires_grad_(True)
    bias = bucket_bias(table, edges, pos, pos[:, :0], member)
    assert not bias.any()
    assert not torch.autograd.grad(bias.sum(), table)[0].any()
