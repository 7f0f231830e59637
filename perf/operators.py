"""Timed cases of the encoder block's operators: the root-mean-square norm with the residual's addition
(16-bit or e4m3 output), the matrix product with bias, activation and residual in its epilogue (16-bit,
32-bit or e4m3 operands) and the bucketed relative-position bias.

``run`` computes a case in plain torch operations, in 32 bits, or, with ``own`` set, through
``affmae_b200.kernels``; ``exact`` gives the same outputs from the definition in 64 bits.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}
E4M3_MAX = 448.0


# ------------------------------------------------------------------ cases --

def listed():
    return [
        # the encoder's first stage at 16 images of 1024 x 1024: 96 -> 192 channels, one training step
        dict(name="linear train stage 1 up", op="linear", rows=524288, k=96, n=192, dtype="bf16", act="gelu",
             residual="", train=True),
        # the decoder's feed-forward network on its 524288 masked queries (the largest product of the model)
        dict(name="linear train decoder up", op="linear", rows=524288, k=384, n=768, dtype="bf16", act="relu",
             residual="", train=True),
        # stage 4's second MLP product for a single token
        dict(name="linear one token", op="linear", rows=1, k=1024, n=512, dtype="bf16", act="none", residual="bf16",
             train=False),
        # stage 3 of one image (5243 tokens): second MLP product added to the fp32 residual stream
        dict(name="linear stage 3 down", op="linear", rows=5243, k=768, n=384, dtype="bf16", act="none",
             residual="fp32", train=False),
        # outside autocast, in 32 bits, odd sizes
        dict(name="linear fp32 odd", op="linear", rows=13107, k=385, n=771, dtype="fp32", act="gelu", residual="",
             train=False),
        # 8-bit operands, one token through a wide layer
        dict(name="linear e4m3 one token", op="linear8", rows=1, k=4096, n=8192, out="bf16", act="none", residual=""),
        # 8-bit operands, a batch through a wide layer
        dict(name="linear e4m3 batch", op="linear8", rows=8192, k=4096, n=8192, out="bf16", act="gelu", residual=""),
        # stage 1 pre-norm in training: fp32 stream, 16-bit branch, stochastic depth per image
        dict(name="norm train stage 1", op="norm", rows=524288, c=96, groups=16, x="fp32", delta="bf16", y="bf16",
             train=True),
        # one token at the last stage's width, 8-bit output
        dict(name="norm e4m3 one token", op="norm8", rows=1, c=512, groups=0, x="bf16", delta="bf16"),
        # wide rows, 8-bit output
        dict(name="norm e4m3 wide", op="norm8", rows=16384, c=4096, groups=0, x="bf16", delta="bf16"),
        # the bias of stage 1's neighbourhood attention: 16 images, 3 heads, 48 neighbours a token
        dict(name="bias train stage 1", op="bias", batch=16, heads=3, nq=32768, nk=32768, m=48, axes=2, edges=7,
             reach=24, one_sided=False, dtype="bf16", train=True),
        # one new token against a long sequence of earlier ones
        dict(name="bias one token", op="bias", batch=8, heads=16, nq=1, nk=65537, m=0, axes=1, edges=31, reach=4096,
             one_sided=True, dtype="fp16", train=False),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "linear", "linear8", "norm", "norm8", "bias", "bias"])
    if op in ("linear", "linear8"):
        while True:
            rows, k, n = _log(rng, 1, 524288), _log(rng, 8, 4096), _log(rng, 8, 8192)
            if rng.random() < 0.6:  # most layers have widths in multiples of 16
                k, n = 16 * max(1, k // 16), 16 * max(1, n // 16)
            if rows * k * n <= 1.5e11 and rows * (k + n) <= 6e8 and 3072 not in (rows, k, n):
                break
        act = rng.choice(["none", "relu", "gelu", "silu"])
        if op == "linear8":
            return dict(op=op, rows=rows, k=k, n=n, out=rng.choice(["bf16", "fp16"]), act=act,
                        residual=rng.choice(["", "same"]))
        dtype = rng.choice(["bf16", "bf16", "fp16", "fp32"])
        return dict(op=op, rows=rows, k=k, n=n, dtype=dtype, act=act, residual=rng.choice(["", "", dtype, "fp32"]),
                    train=rng.random() < 0.5)
    if op in ("norm", "norm8"):
        while True:
            groups, c = rng.choice([0, 0, 2, 16]), _log(rng, 4, 8192)
            rows = _log(rng, 1, 524288 // max(groups, 1)) * max(groups, 1)
            if rng.random() < 0.6:
                c = 8 * max(1, c // 8)
            if rows * c <= 1e8 and 3072 not in (rows, c):
                break
        x = rng.choice(["bf16", "fp16", "fp32"])
        delta = rng.choice(["", x, "bf16"]) if groups == 0 else rng.choice([x, "bf16"])
        if op == "norm8":
            return dict(op=op, rows=rows, c=c, groups=groups, x=x, delta=delta)
        return dict(op=op, rows=rows, c=c, groups=groups, x=x, delta=delta, y=rng.choice([x, "bf16"]),
                    train=rng.random() < 0.7)
    dtype = rng.choice(["bf16", "fp16", "fp32"])
    heads = rng.choice([1, 3, 6, 12, 16])
    if rng.random() < 0.5:  # neighbour lists of clusters of eight tokens
        while True:
            batch, n, m = _log(rng, 1, 16), _log(rng, 64, 32768), 8 * rng.randint(1, 8)
            if batch * n * m * heads <= 8e7 and n != 3072:
                break
        return dict(op=op, batch=batch, heads=heads, nq=n, nk=n, m=m, axes=2, edges=rng.randint(1, 12),
                    reach=rng.choice([16, 24, 64]), one_sided=False, dtype=dtype, train=rng.random() < 0.6)
    while True:
        batch, nq, nk = _log(rng, 1, 16), _log(rng, 1, 4096), _log(rng, 1, 131072)
        if nq <= nk and batch * nq * nk * heads <= 8e7 and 3072 not in (nq, nk):
            break
    return dict(op=op, batch=batch, heads=heads, nq=nq, nk=nk, m=0, axes=1, edges=rng.randint(2, 48),
                reach=rng.choice([128, 1024, 8192]), one_sided=rng.random() < 0.5, dtype=dtype,
                train=rng.random() < 0.5)


def work(case):
    op = case["op"]
    if op in ("linear", "linear8"):
        r, k, n = case["rows"], case["k"], case["n"]
        s = 1 if op == "linear8" else SIZE[case["dtype"]]
        res = _residual_dtype(case)
        o = SIZE[res] if res else SIZE[_out_dtype(case)]
        if op == "linear8":
            b = (r + n) * (k + 4) + 4 * n + r * n * o + (r * n * o if res else 0)
            return dict(bytes=b, flops=2 * r * k * n)
        b = s * (r * k + k * n + n) + r * n * o + (r * n * o if res else 0)
        if not case["train"]:
            return dict(bytes=b, flops=2 * r * k * n)
        return dict(bytes=b + r * n * o + s * (r * k + k * n + n), flops=6 * r * k * n)
    if op in ("norm", "norm8"):
        r, c = case["rows"], case["c"]
        sx = SIZE[case["x"]]
        sd = SIZE[case["delta"]] if case["delta"] else 0
        s_out = sx if sd else 0
        b = r * c * (sx + sd + s_out) + 4 * c + 4 * case["groups"]
        if op == "norm8":
            return dict(bytes=b + r * (c + 4), flops=6 * r * c)
        sy = SIZE[case["y"]]
        b += r * c * sy
        if not case["train"]:
            return dict(bytes=b, flops=5 * r * c)
        return dict(bytes=b + r * c * (sy + s_out + sx + sd) + 4 * c, flops=15 * r * c)
    pairs = case["batch"] * case["nq"] * (case["m"] or case["nk"])
    rows = _table_rows(case)
    p = 4 if case["axes"] == 2 else 8
    b = case["batch"] * (case["nq"] + case["nk"]) * case["axes"] * p + (4 * pairs if case["m"] else 0)
    b += SIZE[case["dtype"]] * (rows * case["heads"] + pairs * case["heads"])
    if case["train"]:
        b += SIZE[case["dtype"]] * (rows * case["heads"] + pairs * case["heads"])
    return dict(bytes=b, flops=pairs * (4 * case["axes"] + case["heads"] * (2 if case["train"] else 1)))


# ----------------------------------------------------------------- inputs --

def _out_dtype(case):
    return case["out"] if case["op"] == "linear8" else case["dtype"]


def _residual_dtype(case):
    return _out_dtype(case) if case["residual"] == "same" else case["residual"]


def _edges(count, reach):
    """Ascending integer distances where a new bucket begins: single steps, then geometric up to `reach`."""
    half = (count + 1) // 2
    e = list(range(1, half + 1))
    for j in range(1, count - half + 1):
        e.append(max(e[-1] + 1, round(half * (max(reach, half) / half) ** (j / (count - half)))))
    return tuple(e)


def _table_rows(case):
    n = case["edges"] + 1 if case["one_sided"] else 2 * case["edges"] + 1
    return n ** case["axes"]


def _clustered(batch, n, m, g):
    """Positions of n tokens kept at random of a square grid, ordered along 4 x 4 cells (so that runs of
    eight are spatial clusters), and each token's list of the members of its m / 8 nearest clusters."""
    side = math.ceil(math.sqrt(2 * n))
    sel = torch.rand((batch, side * side), device="cuda", generator=g).argsort(1)[:, :n]
    x, y = sel % side, sel // side
    order = (((y // 4) * (side // 4 + 1) + x // 4) * 16 + (y % 4) * 4 + x % 4).argsort(1)
    pos = torch.stack([x, y], -1).gather(1, order[..., None].expand(-1, -1, 2)).float()
    clusters, want = max(1, n // 8), m // 8
    mean = pos[:, :clusters * 8].view(batch, clusters, 8, 2).mean(2)
    lists = [torch.cdist(p, c).topk(min(want, clusters), largest=False).indices for p, c in zip(pos, mean)]
    near = torch.stack(lists)
    near = near.repeat(1, 1, -(-want // near.shape[-1]))[..., :want]
    member = (near[..., None] * 8 + torch.arange(8, device="cuda")).reshape(batch, n, m)
    return pos, member.to(torch.int32)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def normal(*shape, std=1.0, dtype=torch.float32):
        return (torch.randn(shape, device="cuda", generator=g) * std).to(dtype)

    def uniform(*shape, bound, dtype=torch.float32):
        return ((torch.rand(shape, device="cuda", generator=g) * 2 - 1) * bound).to(dtype)

    op = case["op"]
    st = dict(case=case)
    if op in ("linear", "linear8"):
        r, k, n = case["rows"], case["k"], case["n"]
        t, res = DTYPES[_out_dtype(case)], _residual_dtype(case)
        st["bias"] = normal(n, std=0.1, dtype=torch.float32 if op == "linear8" else t)
        st["residual"] = normal(r, n, dtype=DTYPES[res]) if res else None
        if op == "linear8":  # operands as a program holds them: e4m3 values and one fp32 scale a row
            st["x"], st["x_scale"] = _to_e4m3(normal(r, k))
            st["w"], st["w_scale"] = _to_e4m3(uniform(n, k, bound=math.sqrt(6 / (k + n))))
            return st
        st["x"] = normal(r, k, dtype=t)
        st["w"] = uniform(n, k, bound=math.sqrt(6 / (k + n)), dtype=t)
        if case["train"]:
            st["dout"] = normal(r, n, std=0.01, dtype=DTYPES[res] if res else t)
            for name in ("x", "w", "bias", "residual"):
                if st[name] is not None:
                    st[name].requires_grad_(True)
        return st
    if op in ("norm", "norm8"):
        r, c = case["rows"], case["c"]
        st["x"] = normal(r, c, std=1.5, dtype=DTYPES[case["x"]])
        st["w"] = 1 + normal(c, std=0.1)
        st["delta"] = normal(r, c, std=0.5, dtype=DTYPES[case["delta"]]) if case["delta"] else None
        # stochastic depth: a group's branch is dropped, or scaled by 1 / keep
        st["factor"] = (torch.rand(case["groups"], device="cuda", generator=g) < 0.9).float() / 0.9 \
            if case["groups"] else None
        if op == "norm" and case["train"]:
            st["dy"] = normal(r, c, std=0.01, dtype=DTYPES[case["y"]])
            st["ds"] = normal(r, c, std=0.01, dtype=DTYPES[case["x"]]) if case["delta"] else None
            for name in ("x", "w", "delta"):
                if st[name] is not None:
                    st[name].requires_grad_(True)
        return st
    b, t = case["batch"], DTYPES[case["dtype"]]
    st["edges"] = _edges(case["edges"], case["reach"])
    st["table"] = normal(_table_rows(case), case["heads"], std=0.5, dtype=t)
    if case["axes"] == 2:
        st["q_pos"], st["member"] = _clustered(b, case["nq"], case["m"], g)
        st["k_pos"] = st["q_pos"]
    else:  # the last nq of nk consecutive positions, each sequence with a start of its own
        start = torch.randint(0, 1 << 40, (b, 1, 1), device="cuda", generator=g)
        st["k_pos"] = start + torch.arange(case["nk"], device="cuda")[None, :, None]
        st["q_pos"] = st["k_pos"][:, case["nk"] - case["nq"]:].contiguous()
        st["member"] = None
    if case["train"]:
        st["dout"] = normal(b, case["heads"], case["nq"], case["m"] or case["nk"], std=0.01, dtype=t)
        st["table"].requires_grad_(True)
    return st


# ------------------------------------------------------------- plain forms --

def _to_e4m3(y):
    """Rows as e4m3 values and the fp32 scale that each row's values stand for."""
    scale = y.abs().amax(-1, keepdim=True) / E4M3_MAX
    scale = torch.where(scale == 0, torch.ones_like(scale), scale)
    return (y / scale).to(torch.float8_e4m3fn), scale[..., 0]


def _act(z, act):
    if act == "relu":
        return torch.where(z > 0, z, 0.0)
    if act == "gelu":
        return z * (0.5 * (1 + torch.erf(z * math.sqrt(0.5))))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_grad(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    s = 1 / (1 + torch.exp(-z))
    return s * (1 + z * (1 - s))


def _plain_linear(st):
    case = st["case"]
    x, w, b = st["x"].float(), st["w"].float(), st["bias"].float()
    z = x @ w.t() + b
    y = _act(z, case["act"])
    if st["residual"] is not None:
        y = y + st["residual"].float()
    out = DTYPES[_residual_dtype(case) or case["dtype"]]
    if not case["train"]:
        return dict(y=y.to(out))
    dz = st["dout"].float()
    if case["act"] != "none":
        dz = dz * _act_grad(z, case["act"])
    t = st["x"].dtype
    grads = dict(dx=(dz @ w).to(t), dw=(dz.t() @ x).to(t), db=dz.sum(0).to(t))
    if st["residual"] is not None:
        grads["dres"] = st["dout"]
    return dict(grads, y=y.to(out))


def _plain_linear8(st):
    case = st["case"]
    x = st["x"].float() * st["x_scale"][:, None]
    w = st["w"].float() * st["w_scale"][:, None]
    y = _act(x @ w.t() + st["bias"], case["act"])
    if st["residual"] is not None:
        y = y + st["residual"].float()
    return dict(y=y.to(DTYPES[case["out"]]))


EPS = 1e-6


def _plain_norm(st):
    case = st["case"]
    r, c = case["rows"], case["c"]
    s = st["x"].float()
    f = st["factor"]
    f = f.repeat_interleave(r // f.numel())[:, None] if f is not None else 1.0
    if st["delta"] is not None:
        s = s + f * st["delta"].float()
    rstd = 1 / torch.sqrt((s * s).mean(-1, keepdim=True) + EPS)
    y = s * rstd * st["w"]
    out = dict(s=s.to(st["x"].dtype)) if st["delta"] is not None else {}
    if case["op"] == "norm8":
        out["q"], out["scale"] = _to_e4m3(y)
        return out
    out["y"] = y.to(DTYPES[case["y"]])
    if case["train"]:
        dy = st["dy"].float()
        gy = dy * st["w"]
        dx = rstd * (gy - s * (rstd * rstd) * (gy * s).mean(-1, keepdim=True))
        if st["ds"] is not None:
            dx = dx + st["ds"].float()
            out["ddelta"] = (f * dx).to(st["delta"].dtype)
        out["dx"] = dx.to(st["x"].dtype)
        out["dw"] = (dy * s * rstd).sum(0)
    return out


def _bucket(delta, edges, one_sided):
    edges = torch.tensor(edges, device=delta.device)
    if one_sided:
        return torch.bucketize((-delta).clamp(min=0), edges, right=True)
    return len(edges) + delta.sign() * torch.bucketize(delta.abs(), edges, right=True)


def _plain_bias(st):
    case = st["case"]
    one = case["one_sided"]
    n = len(st["edges"]) + 1 if one else 2 * len(st["edges"]) + 1
    kp = st["k_pos"]
    if st["member"] is not None:
        b, nq, m = st["member"].shape
        kp = kp.gather(1, st["member"].long().view(b, -1, 1).expand(-1, -1, kp.shape[-1])).view(b, nq, m, -1)
    else:
        kp = kp[:, None]
    row = None
    for axis in reversed(range(case["axes"])):
        i = _bucket(torch.round(kp[..., axis] - st["q_pos"][:, :, None, axis]).long(), st["edges"], one)
        row = i if row is None else row * n + i
    bias = st["table"].detach()[row].permute(0, 3, 1, 2).contiguous()
    if not case["train"]:
        return dict(bias=bias)
    h = case["heads"]
    dtable = torch.zeros((_table_rows(case), h), device="cuda")
    dtable.index_add_(0, row.reshape(-1), st["dout"].permute(0, 2, 3, 1).reshape(-1, h).float())
    return dict(bias=bias, dtable=dtable.to(st["table"].dtype))


# -------------------------------------------------- the framework's kernels --

def _grads(y, of):
    """A linear case's output and its gradients by autograd."""
    names = [("dx", "x"), ("dw", "w"), ("db", "bias")] + ([("dres", "residual")] if of.get("residual") is not None else [])
    grads = torch.autograd.grad(y, [of[n] for _, n in names], of["dout"])
    return dict(zip([d for d, _ in names], grads), y=y.detach())


def _own_linear(st):
    from affmae_b200.kernels.linear import fused_linear
    case = st["case"]
    if not case["train"]:
        with torch.no_grad():
            return dict(y=fused_linear(st["x"], st["w"], st["bias"], act=case["act"], residual=st["residual"]))
    y = fused_linear(st["x"], st["w"], st["bias"], act=case["act"], residual=st["residual"])
    return _grads(y, st)


def _own_linear8(st):
    from affmae_b200.kernels.linear import linear_e4m3
    case = st["case"]
    return dict(y=linear_e4m3(st["x"], st["x_scale"], st["w"], st["w_scale"], st["bias"], act=case["act"],
                              residual=st["residual"], out_dtype=DTYPES[case["out"]]))


def _own_norm(st):
    from affmae_b200.kernels.rms_norm import fused_rms_norm, rms_norm_e4m3
    case = st["case"]
    has_delta = st["delta"] is not None
    if case["op"] == "norm8":
        got = rms_norm_e4m3(st["x"], st["w"], EPS, delta=st["delta"], row_scale=st["factor"])
        return dict(s=got[0], q=got[1], scale=got[2]) if has_delta else dict(q=got[0], scale=got[1])
    with torch.set_grad_enabled(case["train"]):
        got = fused_rms_norm(st["x"], st["w"], EPS, delta=st["delta"], row_scale=st["factor"],
                             out_dtype=DTYPES[case["y"]])
    if has_delta:
        out = dict(s=got[0].detach(), y=got[1].detach())
    else:
        out = dict(y=got.detach())
    if case["train"]:
        if has_delta:
            out["dx"], out["dw"], out["ddelta"] = torch.autograd.grad(got, (st["x"], st["w"], st["delta"]),
                                                                      (st["ds"], st["dy"]))
        else:
            out["dx"], out["dw"] = torch.autograd.grad(got, (st["x"], st["w"]), st["dy"])
    return out


def _own_bias(st):
    from affmae_b200.kernels.bucket_bias import bucket_bias
    case = st["case"]
    with torch.set_grad_enabled(case["train"]):
        bias = bucket_bias(st["table"], st["edges"], st["q_pos"], st["k_pos"], st["member"],
                           one_sided=case["one_sided"])
    if not case["train"]:
        return dict(bias=bias)
    (dtable,) = torch.autograd.grad(bias, (st["table"],), st["dout"])
    return dict(bias=bias.detach(), dtable=dtable)


PLAIN = dict(linear=_plain_linear, linear8=_plain_linear8, norm=_plain_norm, norm8=_plain_norm, bias=_plain_bias)
OWN = dict(linear=_own_linear, linear8=_own_linear8, norm=_own_norm, norm8=_own_norm, bias=_own_bias)


def run(state):
    op = state["case"]["op"]
    if own:
        return OWN[op](state)
    with torch.no_grad():
        return PLAIN[op](state)


# ------------------------------------------------------------------ 64 bits --

def _round_e4m3(v):
    """64-bit values rounded to the nearest e4m3 value (ties to even, steps of 2^-9 below 2^-6, at most 448)."""
    _, e = torch.frexp(v)
    step = torch.exp2((e - 1).clamp(min=-6).double() - 3)
    return (torch.round(v / step) * step).clamp(-E4M3_MAX, E4M3_MAX)


def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    leaf = {k: v.detach().double().requires_grad_(True) for k, v in st.items()
            if torch.is_tensor(v) and v.is_floating_point() or torch.is_tensor(v) and v.dtype == torch.float8_e4m3fn}
    act = dict(none=lambda v: v, relu=torch.nn.functional.relu, gelu=torch.nn.functional.gelu,
               silu=torch.nn.functional.silu)
    if op in ("linear", "linear8"):
        if op == "linear8":
            z = torch.nn.functional.linear(leaf["x"], leaf["w"]) * leaf["x_scale"][:, None] * leaf["w_scale"]
            z = z + leaf["bias"]
        else:
            z = torch.nn.functional.linear(leaf["x"], leaf["w"], leaf["bias"])
        y = act[case["act"]](z)
        if "residual" in leaf:
            y = y + leaf["residual"]
        if op == "linear8" or not case["train"]:
            return dict(y=y.detach())
        return _grads(y, leaf)
    if op in ("norm", "norm8"):
        s = leaf["x"]
        if "delta" in leaf:
            d = leaf["delta"]
            if "factor" in leaf:
                g = leaf["factor"].numel()
                d = (d.view(g, -1) * leaf["factor"].detach()[:, None]).view(s.shape)
            s = s + d
        y = s * torch.rsqrt(s.square().mean(1, keepdim=True) + EPS) * leaf["w"]
        out = dict(s=s.detach()) if "delta" in leaf else {}
        if op == "norm8":
            y = y.detach()
            top = y.abs().max(1).values
            out["scale"] = torch.where(top > 0, top / E4M3_MAX, 1.0)
            out["q"] = _round_e4m3(y / out["scale"][:, None])
            return out
        out["y"] = y.detach()
        if case["train"]:
            if "delta" in leaf:
                out["dx"], out["dw"], out["ddelta"] = torch.autograd.grad(
                    (s, y), (leaf["x"], leaf["w"], leaf["delta"]), (leaf["ds"], leaf["dy"]))
            else:
                out["dx"], out["dw"] = torch.autograd.grad(y, (leaf["x"], leaf["w"]), leaf["dy"])
        return out
    # bias: a table of the bucket of every distance up to the last edge, counted edge by edge
    edges = st["edges"]
    near = torch.zeros(edges[-1] + 1, dtype=torch.long, device="cuda")
    for e in edges:
        near[e:] += 1
    b, nq, m = case["batch"], case["nq"], case["m"] or case["nk"]
    rows, h = _table_rows(case), case["heads"]
    out, dtable = [], torch.zeros((h, rows), dtype=torch.float64, device="cuda")
    for i in range(b):  # one sequence at a time
        kp = st["k_pos"][i]
        kp = kp[st["member"][i].long()] if st["member"] is not None else kp[None].expand(nq, -1, -1)
        row = torch.zeros((nq, m), dtype=torch.long, device="cuda")
        for axis in range(case["axes"]):
            d = (kp[..., axis] - st["q_pos"][i, :, None, axis]).long()
            far = near[d.abs().clamp(max=edges[-1])]
            if case["one_sided"]:
                j, n = torch.where(d < 0, far, 0), len(edges) + 1
            else:
                j, n = torch.where(d < 0, len(edges) - far, len(edges) + far), 2 * len(edges) + 1
            row += j * n ** axis
        out.append(leaf["table"].detach().t()[:, row])
        if case["train"]:
            for k in range(h):
                dtable[k] += torch.bincount(row.reshape(-1), leaf["dout"][i, k].detach().reshape(-1), rows)
    if not case["train"]:
        return dict(bias=torch.stack(out))
    return dict(bias=torch.stack(out), dtable=dtable.t().contiguous())
