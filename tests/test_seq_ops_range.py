"""The sequence operators over the range that they are documented for."""
import pytest
import torch

from tests import seq_reference as R
from tests.test_seq_ops import _gen

BF, FP = torch.bfloat16, torch.float32


# ---------------------------------------------------------------------- gradients of large and small rows of a norm
@pytest.mark.gpu
@pytest.mark.parametrize("dtype,rows,hidden", [(FP, 5, 100), (BF, 9, 1000), (FP, 3, 8196), (BF, 2, 16392)])
@pytest.mark.parametrize("size,eps", [(1e13, 1e-5), (1e15, 1e-5), (3e16, 1e-5), (1e-15, 1e-36)])
def test_norm_gradients_of_large_and_small_rows(dtype, rows, hidden, size, eps):
    """Rows whose rsqrt is far from 1, its cube outside fp32: the squares' sum and every factor of the definition are inside."""
    from silent_speech_amd import ops
    g = _gen(hidden + rows)
    x, dh = (torch.randn(rows, hidden, generator=g) * size).to(dtype), torch.randn(rows, hidden, generator=g).to(dtype)
    dh = (dh.float() + 2.0 * torch.sign(x.float())).to(dtype)  # a gradient along the row: the projection counts
    w = (1 + 0.3 * torch.randn(hidden, generator=g)).to(dtype)
    xd, wd = x.cuda().requires_grad_(), w.cuda().requires_grad_()
    x_out, h = ops.add_rms_norm(xd, None, wd, eps)
    want = R.add_rms_norm(x, None, w, eps, None, dh)
    R.within(h, want["h"], "h")
    dx, dw = torch.autograd.grad(h, (xd, wd), dh.cuda())
    R.within(dx, want["dx"], "dx")
    R.within(dw, want["dw"], "dw")
