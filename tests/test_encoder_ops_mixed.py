"""The encoder-block operators where rows, gradients or callers differ strongly
from one another: rows of other sizes in turn, gradients of mixed magnitude,
infinities, forward-mode derivatives, several threads.  Bounds as in
test_encoder_ops.py."""
import pytest
import torch

from affmae_b200.kernels.linear import quantize_e4m3
from test_encoder_ops import BF16, FP16, FP32, check_e4m3, rnd


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
