"""The encoder-block operators where rows, gradients or callers differ strongly
from one another: rows of other sizes in turn, gradients of mixed magnitude,
infinities, forward-mode derivatives, several threads.  Bounds as in
test_encoder_ops.py."""
import ctypes
import subprocess
import sys
import threading

import pytest
import torch
import torch.autograd.forward_ad as fwAD

from affmae_b200 import _native as nat
from affmae_b200.kernels.bucket_bias import bucket_bias, bucket_count, log_edges
from affmae_b200.kernels.linear import LinearE4M3, fused_linear, linear_e4m3, linear_status, quantize_e4m3
from affmae_b200.kernels.rms_norm import fused_rms_norm, rms_norm_e4m3
from conftest import ROOT
from test_encoder_ops import BF16, E, FP16, FP32, TINY, U, bias_inputs, check_e4m3, linear_ref, rnd, rows_ref, within


@pytest.mark.gpu
@pytest.mark.parametrize("dtype,shape", [(FP32, (5000, 4096)), (FP32, (8192, 1032)), (BF16, (3000, 1025)),
                                         (BF16, (1500, 2048)), (FP16, (6000, 129)), (FP32, (2500, 8200)),
                                         (BF16, (2400, 9000))])
def test_quantize_e4m3_of_several_rows_a_block(cuda, dtype, shape):
    """Rows that a whole block shares, more of them than there are blocks, each of another size than the one before
    it in its block: every value is scaled by its own row's maximum.  Twice, to the same bits."""
    R, C = shape
    size = torch.randint(-6, 7, (R, 1), generator=torch.Generator().manual_seed(1)).to(cuda)
    x = (rnd(cuda, 2, R, C) * torch.exp2(size.float())).to(dtype)
    q, scale = quantize_e4m3(x)
    for i in range(0, R, 1000):
        xd = x[i:i + 1000].double()
        check_e4m3(q[i:i + 1000], scale[i:i + 1000], xd, torch.zeros_like(xd))
    again = quantize_e4m3(x)
    assert torch.equal(q.view(torch.uint8), again[0].view(torch.uint8)) and torch.equal(scale, again[1])


WIDE = [  # B, H, Nq, Nk, M (0: all keys), axes, edges, one sided, position type
    (2, 3, 2000, 2000, 48, 2, log_edges(7, 24), False, FP32),
    (1, 5, 700, 700, 13, 2, (1, 4), False, torch.int32),
    (2, 4, 33, 1001, 0, 1, log_edges(31, 512), True, torch.int64),
    (1, 2, 400, 400, 64, 2, log_edges(32, 60), False, FP32),     # 65 x 65 rows
]


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("case", WIDE)
@pytest.mark.parametrize("kind", ["spread", "outlier", "tiny", "huge"])
def test_bucket_bias_gradients_of_mixed_size(cuda, dtype, case, kind):
    """Every row of the table's gradient against its own terms, whatever the others are: a term is summed exactly
    in integers within a tile; a tile's sum is formed of two to sixteen such sums, and up to eight tiles' and
    blocks' sums are added one after the other, 32 additions in all."""
    B, H, Nq, Nk, M, A, edges, one, _ = case
    qp, kp, member = bias_inputs(cuda, case)
    rows = bucket_count(edges, A, one)
    table = torch.zeros((rows, H), device=cuda, dtype=dtype, requires_grad=True)
    bias = bucket_bias(table, edges, qp, kp, member, one)
    g = torch.Generator().manual_seed(7)
    d = torch.randn(bias.shape, generator=g).double() * 10.0 ** (-8 * torch.rand(bias.shape, generator=g).double())
    if kind == "outlier":
        d = d * 1e-6
        d[0, 0, 0, 0], d[-1, -1, -1, -1] = 3.0, -1e4
    elif dtype != FP16 and kind != "spread":
        d = d * (1e-34 if kind == "tiny" else 1e34)
    dout = d.to(dtype).to(cuda)
    (dt,) = torch.autograd.grad(bias, (table,), dout, retain_graph=True)
    (again,) = torch.autograd.grad(bias, (table,), dout)
    assert torch.equal(dt, again)
    row = rows_ref(edges, qp, kp, member, one).reshape(-1)
    ok = row >= 0
    gd = dout.double().permute(0, 2, 3, 1).reshape(-1, H)[ok]
    ref = torch.zeros((rows, H), dtype=torch.float64, device=cuda).index_add_(0, row[ok], gd)
    mag = torch.zeros_like(ref).index_add_(0, row[ok], gd.abs())
    # 2^-149: fp32's spacing next to zero (bf16's: 2^-133)
    within(dt, ref, 32 * E * mag + U[dtype] * ref.abs() + TINY[dtype] + (2.0 ** -133 if dtype == BF16 else 32 * 2.0 ** -149))


@pytest.mark.gpu
def test_threads_that_launch_one_kernel_with_different_shared_memory(cuda):
    """The norm with and without a residual branch and the bias gradient with two tables, each from a thread of its
    own, each pair through one kernel: no launch depends on what another thread has asked for.  The library is
    called directly, so that the threads are in it together."""
    lib = nat.lib()
    x, d, w = rnd(cuda, 1, 1800, 8192, dtype=BF16), rnd(cuda, 2, 1800, 8192, dtype=BF16), torch.ones(8192, device=cuda)
    pos, dout = rnd(cuda, 3, 1, 8, 2, std=20.0), rnd(cuda, 4, 1, 4, 8, 8)
    y, s = torch.empty_like(x), torch.empty_like(x)
    ws = torch.empty(1 << 20, device=cuda, dtype=torch.uint8)
    out = torch.empty((4225, 4), device=cuda)
    streams = [torch.cuda.Stream() for _ in range(4)]
    jobs = []
    for k, delta in enumerate((None, d)):
        jobs.append((lib.affb_rms_norm_fwd, (x.data_ptr(), 2, nat.ptr(delta), 2, None, 0, w.data_ptr(), 1e-6, 1800, 8192,
                                             s.data_ptr() if k else None, None, y.data_ptr(), 2, None, None,
                                             streams[k].cuda_stream)))
    for k, n in enumerate((20, 32)):
        e = (ctypes.c_int32 * n)(*log_edges(n, 9000))
        jobs.append((lib.affb_bucket_bias_bwd, (dout.data_ptr(), 0, ctypes.addressof(e), n, 0, pos.data_ptr(), pos.data_ptr(),
                                                0, 2, None, 1, 4, 8, 8, 8, out.data_ptr(), 0, ws.data_ptr(), ws.numel(),
                                                streams[2 + k].cuda_stream)))
        jobs[-1] += (e,)
    errors = []

    def work(f, args, stream, *_):
        for i in range(4000):
            if f(*args) != 0:
                errors.append(lib.affb_last_error().decode())
            if i % 100 == 99:
                stream.synchronize()
    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(j[0], j[1], s)) for j, s in zip(jobs, streams)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, f"{len(errors)} calls failed: {errors[0]}"


# ---------------------------------------------------- forward-mode -------

@pytest.mark.gpu
def test_forward_mode_is_refused(cuda):
    """No operator has a forward-mode derivative: a tangent is refused, with and without a gradient asked for, by the
    functions and by the dispatcher's operators; what has no tangent still runs inside a level."""
    import affmae_b200.ops  # noqa: F401
    ops = torch.ops.affb200
    x, w, d = rnd(cuda, 1, 40, 24), rnd(cuda, 2, 16, 24), rnd(cuda, 3, 40, 24)
    table, pos, ones = rnd(cuda, 4, 25, 3), rnd(cuda, 5, 1, 6, 2, std=3.0), torch.ones(24, device=cuda)
    calls = [(lambda t: fused_linear(t, w), x), (lambda t: fused_linear(x, t, act="gelu"), w),
             (lambda t: fused_linear(x, w, t), rnd(cuda, 6, 16)),
             (lambda t: fused_linear(x, w, None, "none", t), rnd(cuda, 7, 40, 16)),
             (lambda t: fused_rms_norm(t, ones), x), (lambda t: fused_rms_norm(x, t), ones),
             (lambda t: fused_rms_norm(x, ones, delta=t)[0], d),
             (lambda t: bucket_bias(t, (1, 3), pos, pos), table),
             (lambda t: ops.linear_fwd(t, w, None, "none", None)[0], x),
             (lambda t: ops.rms_norm_fwd(x, ones, 1e-6, t, None, FP32)[0], d),
             (lambda t: ops.bucket_bias_fwd(t, [1, 3], pos, pos, None, False, FP32), table)]
    for f, t in calls:
        want = f(t)
        with fwAD.dual_level():
            assert torch.equal(f(t), want)
            for leaf in (t, t.clone().requires_grad_(True)):
                with pytest.raises((NotImplementedError, RuntimeError), match="jvp|forward-mode|forward mode"):
                    f(fwAD.make_dual(leaf, torch.ones_like(t)))
        assert torch.equal(f(t), want)


# ------------------------------------------------- 8-bit operands --------

@pytest.mark.gpu
def test_eight_bit_operators_refuse_a_gradient(cuda):
    """Their outputs do not pass for constants: asking for a gradient is refused, also of the residual stream that the
    norm returns, of a residual added to the product, and in forward mode; under no_grad nothing is recorded."""
    x, w, d = (rnd(cuda, i, 40, 32).requires_grad_(True) for i in (1, 2, 3))
    ones, b = torch.ones(32, device=cuda, requires_grad=True), torch.zeros(40, device=cuda, requires_grad=True)
    res = rnd(cuda, 4, 40, 40).requires_grad_(True)
    with torch.no_grad():
        q, sc = quantize_e4m3(x)
        wq, ws = quantize_e4m3(w)
        want = rms_norm_e4m3(x, ones, delta=d)
    assert not any(t.requires_grad for t in (q, sc, *want))
    outs = [quantize_e4m3(w)[1], *rms_norm_e4m3(x, ones, delta=d)[::2], rms_norm_e4m3(x.detach(), ones)[1],
            rms_norm_e4m3(x.detach(), ones.detach(), delta=d)[0], linear_e4m3(q, sc, wq, ws, b),
            linear_e4m3(q, sc, wq, ws, None, "none", res), linear_e4m3(q, sc, *quantize_e4m3(w))]
    for out in outs:
        with pytest.raises(RuntimeError, match="no gradient"):
            out.float().sum().backward()
    assert all(t.grad is None for t in (x, w, d, ones, b, res))
    for p, r in zip(rms_norm_e4m3(x, ones, delta=d), want):
        assert torch.equal(p.detach().float(), r.float())
    with fwAD.dual_level():
        t = fwAD.make_dual(x.detach(), torch.ones_like(x))
        for f in (lambda: quantize_e4m3(t), lambda: rms_norm_e4m3(t, ones.detach())):
            with pytest.raises((NotImplementedError, RuntimeError), match="jvp|forward-mode|forward mode"):
                f()
    layer = LinearE4M3(w, b)
    assert not any(t.requires_grad for t in layer.state_dict().values())


@pytest.mark.gpu
def test_quantised_block_refuses_a_gradient(cuda):
    from test_rms_block import _block, _inputs
    blk = _block(cuda).eval().quantize()
    pos, member, mask, feat = _inputs(cuda)
    with torch.no_grad():
        want, _ = blk(feat, member, mask, pos)
    got, _ = blk(feat, member, mask, pos)
    assert torch.equal(got.detach(), want)
    with pytest.raises(RuntimeError, match="no gradient"):
        got.sum().backward()


@pytest.mark.gpu
def test_quantised_block_answers_with_the_weights_it_has(cuda):
    """After a change of the weights by any way, a quantised block answers as one that is quantised then; its state
    is that of the block itself."""
    from test_rms_block import _block, _inputs
    pos, member, mask, feat = _inputs(cuda)
    blk, other = _block(cuda).eval(), _block(cuda, seed=9).eval()
    names = list(blk.state_dict())
    blk.quantize()
    assert list(blk.state_dict()) == names
    other.load_state_dict(blk.state_dict())

    def answer(b):
        with torch.no_grad():
            return b(feat, member, mask, pos)[0]

    def in_place(b):
        with torch.no_grad():
            for p in b.parameters():
                p.mul_(1.25)

    def behind(b):
        for p in b.parameters():
            p.data = p.data * 0.5 + 0.01
            p.data.add_(0.01)

    def replaced(b):
        b.fc1.weight = torch.nn.Parameter(b.fc1.weight.detach().flip(0))

    def loaded(b):
        b.load_state_dict({k: v * 0.75 for k, v in _block(cuda, seed=11).state_dict().items()})

    def trained(b):
        b.train()
        b(feat, member, mask, pos)[0].square().mean().backward()
        with torch.no_grad():
            for p in b.parameters():
                p -= 0.1 * p.grad
        b.eval()
    before = answer(blk)
    for change in (in_place, behind, replaced, loaded, trained):
        change(blk)
        change(other)
        got = answer(blk)
        want = answer(other.quantize())
        assert torch.equal(got, want) and not torch.equal(got, before), change.__name__
        before = got
    fresh = _block(cuda, seed=12).eval()
    fresh.load_state_dict(blk.state_dict())
    assert torch.equal(answer(fresh.quantize()), before)


def test_checkpoints_with_the_former_copies_load():
    from affmae_b200.mae import RMSClusterBlock
    blk = torch.nn.Sequential(RMSClusterBlock(8, 1, 2.0, 0.0, (1, 2)))
    state = blk.state_dict()
    blk.load_state_dict({**state, "0.eight_bit.q.weight": torch.zeros(8, 8), "0.eight_bit.q.bias": torch.zeros(8)})
    with pytest.raises(RuntimeError, match="other"):
        blk.load_state_dict({**state, "0.other.q.weight": torch.zeros(8, 8)})


# ---------------------------------------------- waits that run out -------

@pytest.mark.gpu
@pytest.mark.parametrize("name", ["linear", "backward", "few rows", "e4m3", "norm", "norm backward", "quantize"])
def test_a_wait_that_runs_out_is_reported_once(cuda, name):
    """After it (here one of 50 ms that nothing ends, on a stream that blocks no other) the next call raises, and the
    one after that runs; nothing is left behind."""
    x, w = rnd(cuda, 1, 64, 64, dtype=BF16), rnd(cuda, 2, 32, 64, dtype=BF16)
    ones = torch.ones(64, device=cuda)
    q, s = quantize_e4m3(x)
    leaf, vec = x.clone().requires_grad_(True), ones.clone().requires_grad_(True)
    y, n = fused_linear(leaf, w), fused_rms_norm(x, vec)
    f = {"linear": lambda: fused_linear(x, w), "few rows": lambda: fused_linear(x[:2], w),
         "backward": lambda: torch.autograd.grad(y.sum(), leaf, retain_graph=True)[0],
         "e4m3": lambda: linear_e4m3(q, s, q, s), "norm": lambda: fused_rms_norm(x, ones),
         "norm backward": lambda: torch.autograd.grad(n.sum(), vec, retain_graph=True)[0],
         "quantize": lambda: quantize_e4m3(x)[1]}[name]
    want = f()
    assert linear_status()
    stream = torch.cuda.Stream()
    nat.call("affb_linear_wait_probe", 50, stream.cuda_stream)
    stream.synchronize()
    with pytest.raises(RuntimeError, match="bounded wait"):
        f()
    assert torch.equal(f(), want) and linear_status()


@pytest.mark.gpu
def test_status_waits_for_every_stream_and_reports_once(cuda):
    assert linear_status()
    nat.call("affb_linear_wait_probe", 200, torch.cuda.Stream().cuda_stream)
    assert not linear_status()      # without waiting for that stream it would not know yet
    assert linear_status()
    with pytest.raises(RuntimeError, match="limit"):
        nat.call("affb_linear_wait_probe", 0, None)


# ------------------------------------------------ infinities in fp32 -----

def same_class(got, want, what):
    """NaN where `want` (64 bits) is NaN, the same infinity where it is infinite, finite elsewhere."""
    for f in (torch.isnan, torch.isposinf, torch.isneginf):
        assert torch.equal(f(got), f(want)), (what, f.__name__)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [FP32, BF16])
@pytest.mark.parametrize("shape", [(1, 24, 40), (8, 24, 40), (9, 24, 40), (9, 33, 200), (300, 200, 392), (3000, 24, 7)])
@pytest.mark.parametrize("act", ["none", "relu"])
def test_infinities_whatever_the_number_of_rows(cuda, dtype, shape, act):
    """An infinite or NaN operand, gradient or weight gives what the definition gives, from one row to many; the
    rest is as it is without them."""
    M, N, K = shape
    x, w, b = rnd(cuda, 1, M, K, dtype=dtype), rnd(cuda, 2, N, K, dtype=dtype), rnd(cuda, 3, N, dtype=dtype)
    dout = rnd(cuda, 4, M, N, dtype=dtype)
    w[1, 3], w[N - 1, 0] = 0, float("-inf")       # infinity times zero; a whole column of infinities
    x[M // 2, 3] = float("inf")
    x[M - 1, K - 1] = float("-inf") if M > 1 else x[M - 1, K - 1]
    dout[0, 2] = float("inf")
    if M > 2:
        x[1, 0] = float("nan")
        dout[M - 1, 0] = float("nan")
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    ref = [t.double().requires_grad_(True) for t in (x, w, b)]
    y = fused_linear(*leaves, act=act)
    z = ref[0] @ ref[1].T + ref[2]
    yr = z.relu() if act == "relu" else z
    same_class(y.detach(), yr.detach(), "y")
    keep = yr.detach().isfinite()
    tol = (U[dtype] * yr.abs() + (K + 18) * E * (torch.where(x.isfinite(), x, 0).double().abs()
                                                  @ torch.where(w.isfinite(), w, 0).double().abs().T + 8)).detach()
    within(torch.where(keep, y.detach(), 0), torch.where(keep, yr.detach(), 0), torch.where(keep, tol, 1))
    if act == "none":
        for n, p, q in zip("xwb", torch.autograd.grad(y, leaves, dout), torch.autograd.grad(yr, ref, dout.double())):
            same_class(p, q, "d" + n)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP16, FP32])
@pytest.mark.parametrize("shape", [(700, 96), (64, 1000), (5, 8200), (2000, 2048), (33, 7)])
def test_quantize_e4m3_is_its_definition(cuda, dtype, shape):
    """Bit for bit: the row's maximum over 448 and the quotients, each rounded once to fp32, then to e4m3 (at most
    448); rows from the smallest numbers of the type to the largest, zeros, and values on ties."""
    R, C = shape
    x = rnd(cuda, 2, R, C)
    low, high = {BF16: (-133, 126), FP16: (-24, 14), FP32: (-149, 126)}[dtype]
    x = x * torch.exp2(torch.linspace(low, high, R, device=cuda, dtype=torch.float64))[:, None].double()
    x[R // 2] = 0
    x[R // 2 + 1] = torch.randint(-896, 897, (C,), device=cuda) / 2     # whole and half steps of a scale of one
    x[R // 2 + 1, 0] = 448
    x = x.clamp(-torch.finfo(dtype).max, torch.finfo(dtype).max).to(dtype)
    assert x.isfinite().all()
    q, scale = quantize_e4m3(x)
    q, scale, x = q.cpu(), scale.cpu(), x.cpu()
    top = x.float().abs().amax(1)
    want = top / torch.full_like(top, 448)      # on the host, where both are IEEE divisions
    want = torch.where(want == 0, 1.0, want)
    assert torch.equal(scale, want)
    quot = (x.float() / want[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
    assert torch.equal(q.view(torch.uint8), quot.view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP32])
@pytest.mark.parametrize("shape", [(5, 24, 40), (300, 200, 64)])
@pytest.mark.parametrize("with_residual", [False, True])
def test_relu_cuts_off_gradients_that_are_not_finite(cuda, dtype, shape, with_residual):
    """Where ReLU has cut a value off, an infinite or NaN gradient is none: the gradients are those of zeros there."""
    M, N, K = shape
    x, w, b = rnd(cuda, 1, M, K, dtype=dtype), rnd(cuda, 2, N, K, dtype=dtype), rnd(cuda, 3, N, dtype=dtype)
    res = rnd(cuda, 4, M, N, dtype=dtype) if with_residual else None
    dout = rnd(cuda, 5, M, N, dtype=dtype)
    leaves = [t.clone().requires_grad_(True) for t in (x, w, b)]
    y = fused_linear(*leaves, "relu", res)
    off = fused_linear(x, w, b) <= 0
    assert 0 < int(off.sum()) < off.numel()
    bad = torch.where(torch.arange(N, device=cuda) % 2 == 0, float("nan"), float("-inf")).to(dtype).expand(M, N)
    want = torch.autograd.grad(y, leaves, torch.where(off, 0, dout), retain_graph=True)
    got = torch.autograd.grad(y, leaves, torch.where(off, bad, dout))
    assert all(torch.equal(p, q) and p.isfinite().all() for p, q in zip(got, want))


def test_edges_are_taken_by_value():
    """Edges given as tensors or arrays are read at every call."""
    from affmae_b200.kernels.bucket_bias import _check_edges
    edges = [torch.tensor(1), torch.tensor(4)]
    assert _check_edges(edges) == (1, 4) and _check_edges(torch.tensor([1, 4])) == (1, 4)
    edges[1].fill_(6)
    got = _check_edges(edges)
    assert got == (1, 6) and all(type(e) is int for e in got)
    edges[1].fill_(1)
    with pytest.raises(RuntimeError, match="edges"):
        _check_edges(edges)
    assert _check_edges((1.0, 2.0)) == (1, 2) and _check_edges((1, 2)) == (1, 2)


@pytest.mark.gpu
def test_dispatcher_refuses_gradients_of_what_is_kept(cuda):
    """The sums and reciprocal roots that the dispatcher's operators return for the backward have no gradient, and say
    so when one is asked for."""
    import affmae_b200.ops  # noqa: F401
    ops = torch.ops.affb200
    x, w, ones = rnd(cuda, 1, 40, 24).requires_grad_(True), rnd(cuda, 2, 16, 24), torch.ones(24, device=cuda)
    out, z = ops.linear_fwd(x, w, None, "gelu", None)
    s, y, rstd = ops.rms_norm_fwd(x, ones, 1e-6, x.detach(), None, FP32)
    for t in (z, out + z, rstd, y.sum(1) + rstd):
        with pytest.raises(RuntimeError, match="no gradient of its own"):
            t.sum().backward(retain_graph=True)
    assert x.grad is None
    (out.sum() + s.sum() + y.sum()).backward()
    assert x.grad.isfinite().all() and x.grad.any()


@pytest.mark.gpu
def test_dispatcher_computes_what_is_wanted(cuda):
    """Gradients that nothing asks for come back empty from the backward operators, and the others are the same; the
    forward writes no sums without `save`, and then has no gradient."""
    import affmae_b200.ops  # noqa: F401
    ops = torch.ops.affb200
    x, w, b, ones = rnd(cuda, 1, 40, 24), rnd(cuda, 2, 16, 24), rnd(cuda, 3, 16), rnd(cuda, 4, 24)
    dout, ds, d = rnd(cuda, 5, 40, 16), rnd(cuda, 6, 40, 24), rnd(cuda, 7, 40, 24)
    out, z = ops.linear_fwd(x, w, b, "gelu", None)
    bare, none = ops.linear_fwd(x, w, b, "gelu", None, False)
    assert torch.equal(out, bare) and none.numel() == 0 and z.shape == out.shape
    full = ops.linear_bwd(dout, z, x, w, b, "gelu")
    s, y, rstd = ops.rms_norm_fwd(x, ones, 1e-6, d, None, FP32)
    norm = ops.rms_norm_bwd(ds, ds, s, rstd, ones, None, d)
    for i in range(3):
        need = [i == j for j in range(3)]
        got = ops.linear_bwd(dout, z, x, w, b if need[2] else None, "gelu", need[0], need[1])
        assert torch.equal(got[i], full[i]) and sum(t.numel() for t in got) == full[i].numel()
        got = ops.rms_norm_bwd(ds, ds, s, rstd, ones, None, d, *need)
        assert torch.equal(got[i], norm[i]) and sum(t.numel() for t in got) == norm[i].numel()
        leaves = [t.clone().requires_grad_(n) for t, n in zip((x, w, b), need)]
        assert torch.equal(torch.autograd.grad(ops.linear_fwd(*leaves, "gelu", None)[0], leaves[i], dout)[0], full[i])
        leaves = [t.clone().requires_grad_(n) for t, n in zip((x, ones, d), need)]
        got = ops.rms_norm_fwd(leaves[0], leaves[1], 1e-6, leaves[2], None, FP32)
        assert torch.equal(torch.autograd.grad((got[0], got[1]), leaves[i], (ds, ds))[0], norm[i])
    leaf = x.clone().requires_grad_(True)
    with pytest.raises(RuntimeError, match="without save"):
        ops.linear_fwd(leaf, w, b, "gelu", None, False)[0].sum().backward()
    ops.linear_fwd(leaf, w, b, "relu", None, False)[0].sum().backward()   # ReLU's output serves
    assert leaf.grad.any()


@pytest.mark.gpu
@pytest.mark.parametrize("M", [1, 2, 3, 4, 5])
@pytest.mark.parametrize("N,K", [(4096, 1024), (4096, 1040), (2048, 4096), (1200, 4100)])
def test_few_rows_on_both_sides_of_the_rule(cuda, M, N, K):
    """Around the size from which two to four rows go to the tensor cores, 16-bit and e4m3 operands."""
    x, w, b = rnd(cuda, 1, M, K, dtype=BF16), rnd(cuda, 2, N, K, std=K ** -0.5, dtype=BF16), rnd(cuda, 3, N, dtype=BF16)
    out, tol = linear_ref(x, w, b, "gelu", None)
    within(fused_linear(x, w, b, "gelu"), out, tol)
    q, s = quantize_e4m3(x)
    wq, ws = quantize_e4m3(w)
    xd, wd = q.double() * s.double()[:, None], wq.double() * ws.double()[:, None]
    z = xd @ wd.T + b.double()
    zerr = (K + 16) * E * (xd.abs() @ wd.abs().T) + 4 * E * (z.abs() + b.double().abs())
    within(linear_e4m3(q, s, wq, ws, b, out_dtype=FP32), z, zerr + E * z.abs())


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, FP32])
def test_bucket_bias_gradient_of_the_largest_table(cuda, dtype):
    """65 x 65 rows beside the widest table of offsets: a block's whole shared memory."""
    n, m, edges = 100000, 64, tuple(range(1, 32)) + (44,)
    g = torch.Generator().manual_seed(5)
    qp, kp = (torch.randint(0, 100, (1, k, 2), generator=g).float().to(cuda) for k in (n, 4096))
    member = torch.randint(0, 4096, (1, n, m), generator=g).to(cuda, torch.int32)
    table = torch.zeros((65 * 65, 2), device=cuda, dtype=dtype, requires_grad=True)
    dout = rnd(cuda, 6, 1, 2, n, m, dtype=dtype)
    bias = bucket_bias(table, edges, qp, kp, member)
    (dt,) = torch.autograd.grad(bias, (table,), dout)
    row = rows_ref(edges, qp, kp, member, False).reshape(-1)
    gd = dout.double().permute(0, 2, 3, 1).reshape(-1, 2)
    ref = torch.zeros((65 * 65, 2), dtype=torch.float64, device=cuda).index_add_(0, row, gd)
    mag = torch.zeros_like(ref).index_add_(0, row, gd.abs())
    # a block of an SM sums at most 16 tiles' sums, of two or three parts each; then 32 of up to 24 blocks' sums
    within(dt, ref, 128 * E * mag + U[dtype] * ref.abs())


@pytest.mark.gpu
def test_a_captured_graph_may_hold_the_first_call(cuda):
    """The first product and norm of a process may be those that a graph captures."""
    code = """
import torch
from affmae_b200.kernels.linear import fused_linear, linear_status
from affmae_b200.kernels.rms_norm import fused_rms_norm
x, w = torch.randn(300, 64, device="cuda"), torch.randn(32, 64, device="cuda")
ones = torch.ones(64, device="cuda")
torch.cuda.synchronize()
g = torch.cuda.CUDAGraph()
with torch.no_grad(), torch.cuda.graph(g):
    y = fused_linear(fused_rms_norm(x, ones), w, act="gelu")
g.replay()
assert torch.equal(y, fused_linear(fused_rms_norm(x, ones), w, act="gelu")) and linear_status()
print("captured")
"""
    got = subprocess.run([sys.executable, "-c", code], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0 and "captured" in got.stdout, got.stderr[-2000:]
