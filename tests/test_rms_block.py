"""The "rms" encoder block (root-mean-square norms, fused matrix products,
bucketed position bias) against its formula in 64 bits, in the autoencoder,
with 8-bit operands, and its operators through the dispatcher."""
import pytest
import torch
import torch.nn.functional as F

import oracle
from conftest import rel_err

BF16 = torch.bfloat16


def _inputs(dev, B=2, side=16, dim=64, seed=0):
    from affmae_b200.mae import neighbourhood
    from affmae_b200.workloads import clustered_tokens
    pos = clustered_tokens(B, side, 0.5, seed, "cpu").to(dev)
    means = pos.view(B, -1, 8, 2).mean(2)
    member, mask, _ = neighbourhood(pos, means, None, 48, 8)
    g = torch.Generator().manual_seed(seed + 1)
    feat = torch.randn((B, pos.shape[1], dim), generator=g).to(dev)
    return pos, member, mask, feat


def _block(dev, dim=64, heads=2, drop_path=0.0, seed=3):
    from affmae_b200.mae import RMSClusterBlock
    torch.manual_seed(seed)
    blk = RMSClusterBlock(dim, heads, 2.0, drop_path, (1, 2, 3, 5, 9)).to(dev)
    with torch.no_grad():
        for p in blk.parameters():
            if p.dim() == 1:
                p.add_(0.1 * torch.randn_like(p))
        blk.attn.bias.table.normal_(0, 0.5)
    return blk


def _formula(blk, P, feat, member, pos, factors):
    """One block from its definition; P: parameters by name in 64 bits, factors: (attention, MLP) branch factors."""
    def lin(name, x):
        return x @ P[name + ".weight"].T + P[name + ".bias"]

    def norm(name, x):
        return x / (x.square().mean(-1, keepdim=True) + 1e-6).sqrt() * P[name + ".weight"]
    B, N, C = feat.shape
    H, d = blk.attn.heads, C // blk.attn.heads
    h = norm("norm1", feat)
    q = lin("attn.q", h).view(B, N, H, d).transpose(1, 2)
    k, v = lin("attn.kv", h).view(B, N, H, 2, d).permute(3, 0, 2, 1, 4)  # per head: k, then v
    off = pos.gather(1, member.long().view(B, -1, 1).expand(-1, -1, 2)).view(B, N, -1, 2) - pos[:, :, None]
    cnt = sum((off.abs() >= e).long() for e in blk.attn.bias.edges)
    idx = len(blk.attn.bias.edges) + off.sign().long() * cnt
    n = 2 * len(blk.attn.bias.edges) + 1
    bias = P["attn.bias.table"][idx[..., 1] * n + idx[..., 0]].permute(0, 3, 1, 2)
    o = oracle.nbhd_attn_formula(q, k, v, member.cpu(), d ** -0.5, bias=bias, blank_k=P["attn.blank_k"].view(H, d),
                                 blank_v=P["attn.blank_v"].view(H, d))
    x = feat + factors[0] * lin("attn.proj", o.transpose(1, 2).reshape(B, N, C))
    return x + factors[1] * lin("fc2", F.gelu(lin("fc1", norm("norm2", x))))


@pytest.mark.gpu
@pytest.mark.parametrize("drop_path", [0.0, 0.5])
def test_rms_block_matches_its_formula(cuda, drop_path):
    """Forward and every gradient in fp32; the bounds are those of the fp32 attention kernel's own tests (1e-5 / 1e-4
    of the largest value), which the sums of the other operators stay well below."""
    from affmae_b200.mae import add_pending
    blk = _block(cuda, drop_path=drop_path).train()
    pos, member, mask, feat = _inputs(cuda)
    used = []
    if drop_path:
        fixed = [torch.tensor([0.0, 2.0], device=cuda), torch.tensor([2.0, 2.0], device=cuda)]
        blk.drop_path.factor = lambda B, dev: used.append(fixed[len(used)]) or used[-1]
    x = feat.clone().requires_grad_(True)
    out, pending = blk(x, member, mask, pos)
    out = add_pending(out, pending)
    dout = torch.randn(out.shape, generator=torch.Generator().manual_seed(5)).to(cuda)
    names = [n for n, _ in blk.named_parameters()]
    grads = torch.autograd.grad(out, [x] + list(blk.parameters()), dout)
    P = {n: p.detach().cpu().double().requires_grad_(True) for n, p in blk.named_parameters()}
    xr = feat.cpu().double().requires_grad_(True)
    fs = [f.cpu().double().view(-1, 1, 1) for f in used] or [1.0, 1.0]
    ref = _formula(blk, P, xr, member.cpu(), pos.cpu().double(), fs)
    want = torch.autograd.grad(ref, [xr] + list(P.values()), dout.cpu().double())
    assert rel_err(out.detach(), ref.detach()) < 1e-5
    for n, a, b in zip(["feat"] + names, grads, want):
        assert rel_err(a, b) < 1e-4, n


@pytest.mark.gpu
def test_rms_block_under_autocast_and_global(cuda):
    """bf16 autocast against the fp32 block (bf16 operands: 2e-2 of the largest value, as the attention's bf16
    tests), with the residual stream in fp32; the all-pairs form equals lists that name every token."""
    blk = _block(cuda).eval()
    pos, member, mask, feat = _inputs(cuda)
    with torch.no_grad():
        ref, _ = blk(feat, member, mask, pos)
        with torch.autocast("cuda", dtype=BF16):
            out, pending = blk(feat, member, mask, pos)
            again, _ = blk(feat.to(BF16), member, mask, pos)
    assert pending is None and out.dtype == torch.float32 and again.dtype == torch.float32
    assert rel_err(out, ref) < 2e-2
    n = 40
    every = torch.arange(n, device=cuda, dtype=torch.int32).expand(2, n, n).contiguous()
    with torch.no_grad():
        a, _ = blk(feat[:, :n], every, None, pos[:, :n])
        b, _ = blk(feat[:, :n], None, None, pos[:, :n], global_attn=True)
    assert rel_err(a, b) < 1e-5


@pytest.mark.gpu
def test_rms_block_with_eight_bit_operands(cuda):
    """e4m3 operands round each value by up to 2^-4: a projection's error stays below 2 * 2^-4 of its norm
    (independent errors average out over the channels), and so does that of a branch."""
    blk = _block(cuda).eval()
    pos, member, mask, feat = _inputs(cuda)
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16):
        ref, _ = blk(feat, member, mask, pos)
        plain, _ = blk(feat, member, mask, pos)
        out, _ = blk.quantize()(feat, member, mask, pos)
        delta = torch.randn_like(feat).to(BF16)
        f = torch.tensor([1.0, 0.5], device=cuda)
        with_pending, _ = blk(feat, member, mask, pos, pending=(delta, f))
        whole, _ = blk(feat + f.view(2, 1, 1) * delta, member, mask, pos)
    assert torch.equal(ref, plain)
    assert not torch.equal(out, ref) and (out - ref).norm() < 2 * 2.0 ** -4 * (ref - feat).norm()
    assert (with_pending - whole).norm() < 1e-2 * whole.norm()
    blk.train()
    with torch.autocast("cuda", dtype=BF16):
        trained, _ = blk(feat, member, mask, pos)     # training never takes the 8-bit form
    assert (trained - ref).norm() < 1e-2 * ref.norm()


@pytest.mark.gpu
def test_autoencoder_trains_and_answers_with_rms_blocks(cuda):
    from affmae_b200.mae import MAEConfig
    from affmae_b200.pretrain import build, synthetic_images, train_step
    cfg = MAEConfig(img_size=128, embed_dims=(32, 64, 64, 64), depths=(1, 1, 1, 1), num_heads=(1, 2, 2, 2),
                    decoder_dim=64, decoder_heads=2, block="rms")
    model, opt = build(cfg, device=cuda)
    imgs = synthetic_images(2, 128, 0, cuda)
    noise = torch.rand((2, 1024), device=cuda)
    losses = [float(train_step(model, opt, imgs, noise=noise)) for _ in range(6)]
    assert all(l == l for l in losses) and losses[-1] < losses[0]
    model.eval()
    with torch.no_grad(), torch.autocast("cuda", dtype=BF16):
        a, _ = model(imgs, noise=noise)
        b, _ = model.quantize_encoder()(imgs, noise=noise)
    assert abs(float(a) - float(b)) < 0.05 * float(a)
    from affmae_b200.kernels.linear import linear_status
    assert linear_status()


def test_unknown_block_and_quantise_need_rms():
    from affmae_b200.mae import AFFMaskedAutoEncoder, MAEConfig
    small = dict(img_size=64, embed_dims=(8, 8), depths=(1, 1), num_heads=(1, 1), decoder_dim=8, decoder_heads=1)
    with pytest.raises(ValueError, match="block"):
        AFFMaskedAutoEncoder(MAEConfig(block="x", **small))
    with pytest.raises(RuntimeError, match="rms"):
        AFFMaskedAutoEncoder(MAEConfig(**small)).quantize_encoder()


def test_layer_block_parameters_are_what_they_were():
    """The default blocks draw the same initial weights in the same order as before "rms" existed."""
    from affmae_b200.mae import ClusterBlock, MAEConfig, Stage
    cfg = MAEConfig()
    torch.manual_seed(0)
    a = Stage(32, None, 2, 2, cfg, [0.0, 0.1])
    torch.manual_seed(0)
    b = [ClusterBlock(32, 2, cfg.mlp_ratio, dp) for dp in (0.0, 0.1)]
    for x, y in zip(a.blocks.parameters(), torch.nn.ModuleList(b).parameters()):
        assert torch.equal(x, y)


# ------------------------------------------------------------ dispatcher --

def test_block_operators_have_schemas_and_fake_shapes():
    import affmae_b200.ops  # noqa: F401
    from torch._subclasses.fake_tensor import FakeTensorMode
    ops = torch.ops.affb200
    with FakeTensorMode():
        x, w = torch.empty((3, 5, 8), dtype=BF16), torch.empty((6, 8), dtype=BF16)
        res = torch.empty((3, 5, 6))
        out, z = ops.linear_fwd(x, w, None, "gelu", res)
        assert out.shape == (3, 5, 6) and out.dtype == torch.float32 and z.shape == out.shape and z.dtype == torch.float16
        assert ops.linear_fwd(x, w, None, "relu", None)[1].numel() == 0
        dx, dw, db = ops.linear_bwd(out, z, x, w, None, "gelu")
        assert dx.shape == x.shape and dw.shape == w.shape and db.numel() == 0
        s, y, rstd = ops.rms_norm_fwd(x, torch.empty(8), 1e-6, x, None, torch.float32)
        assert s.dtype == BF16 and y.dtype == torch.float32 and rstd.shape == (15,)
        s, q, scale = ops.rms_norm_e4m3(x, torch.empty(8), 1e-6, None, None)
        assert s.numel() == 0 and q.dtype == torch.float8_e4m3fn and scale.shape == (3, 5)
        assert ops.linear_e4m3(q, scale, q[0], scale[0], None, "none", None, BF16).shape == (3, 5, 5)
        b = ops.bucket_bias_fwd(torch.empty((25, 4)), [1, 3], torch.empty((2, 7, 2)), torch.empty((2, 9, 2)), None, False,
                                BF16)
        assert b.shape == (2, 4, 7, 9) and b.dtype == BF16


@pytest.mark.gpu
def test_block_operators_through_the_dispatcher(cuda):
    import affmae_b200.ops  # noqa: F401
    from affmae_b200.kernels.bucket_bias import bucket_bias
    from affmae_b200.kernels.linear import fused_linear, linear_e4m3
    from affmae_b200.kernels.rms_norm import fused_rms_norm, rms_norm_e4m3
    ops = torch.ops.affb200
    g = torch.Generator().manual_seed(0)
    x, w, b, r, d = (torch.randn(s, generator=g).to(cuda) for s in ((40, 24), (16, 24), (16,), (40, 16), (40, 24)))

    def leaves(*ts):
        return [t.clone().requires_grad_(True) for t in ts]
    for act, res in (("gelu", r), ("relu", None), ("none", None), ("silu", None)):
        one, two = leaves(x, w, b), leaves(x, w, b)
        y1 = ops.linear_fwd(*one, act, res)[0]
        y2 = fused_linear(*two, act, res)
        assert torch.equal(y1, y2)
        for p, q in zip(torch.autograd.grad(y1, one, r), torch.autograd.grad(y2, two, r)):
            assert torch.equal(p, q)
    wn = torch.rand(24, generator=g).to(cuda)
    one, two = leaves(x, wn, d), leaves(x, wn, d)
    s1, y1, _ = ops.rms_norm_fwd(one[0], one[1], 1e-6, one[2], None, torch.float32)
    s2, y2 = fused_rms_norm(two[0], two[1], 1e-6, two[2])
    assert torch.equal(s1, s2) and torch.equal(y1, y2)
    for p, q in zip(torch.autograd.grad((s1, y1), one, (x, d)), torch.autograd.grad((s2, y2), two, (x, d))):
        assert torch.equal(p, q)
    one, two = leaves(x, wn), leaves(x, wn)
    y1 = ops.rms_norm_fwd(one[0], one[1], 1e-6, None, None, torch.float32)[1]
    for p, q in zip(torch.autograd.grad(y1, one, d), torch.autograd.grad(fused_rms_norm(*two), two, d)):
        assert torch.equal(p, q)
    _, q, sc = ops.rms_norm_e4m3(x, wn, 1e-6, None, None)
    q2, sc2 = rms_norm_e4m3(x, wn)
    assert torch.equal(q.view(torch.uint8), q2.view(torch.uint8)) and torch.equal(sc, sc2)
    assert torch.equal(ops.linear_e4m3(q, sc, q[:8], sc[:8], None, "gelu", None, BF16),
                       linear_e4m3(q, sc, q[:8], sc[:8], None, "gelu"))
    pos = torch.rand((2, 20, 2), generator=g).to(cuda) * 10
    t1, t2 = leaves(torch.randn((25, 4), generator=g).to(cuda), ) + leaves(torch.zeros((25, 4), device=cuda))
    t2.data.copy_(t1.data)
    b1 = ops.bucket_bias_fwd(t1, [1, 3], pos, pos, None, False, torch.float32)
    b2 = bucket_bias(t2, (1, 3), pos, pos)
    assert torch.equal(b1, b2)
    assert torch.equal(torch.autograd.grad(b1.sum(), t1)[0], torch.autograd.grad(b2.sum(), t2)[0])
