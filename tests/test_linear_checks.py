"""The gradient check of linear_checks by itself, on formulas in 64 bits with x and the weights rounded to fp16 as the kernels round them:
right gradients pass, wrong ones do not."""
import pytest
import torch

import oracle as O
from linear_checks import DIFFERENCE, along_errors, directions, off_the_kink, wrong
from linear_ref import act_grad


def to_fp16(t):
    """fp16 after a power of two per row."""
    s = torch.exp2(14 - t.abs().amax(-1, keepdim=True).log2().floor())
    return (t * s).half().double() / s


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("fmt", [O.Q8_0, O.Q4_K])
def test_wrong_gradients_miss(act, fmt):
    m, n, k = 24, 96, 256
    w = torch.from_numpy(O.dequant(fmt, O.gen_weights(fmt, n, k, seed=9018)).reshape(n, k)).double()
    gen = torch.Generator().manual_seed(18)
    x = (torch.randn(m, k, generator=gen) * 1.5 / (float(w.pow(2).mean().sqrt()) * k ** 0.5)).double()
    bias, dy = 0.5 * torch.randn(n, generator=gen).double(), 0.1 * torch.randn(m, n, generator=gen).double()
    w16 = to_fp16(w)
    z = x @ w.t() + bias
    dy = off_the_kink(act, z, dy)

    def loss_x(x):
        return float((act_grad(act, to_fp16(x) @ w16.t() + bias)[0] * dy).sum())

    def loss_b(b):
        return float((act_grad(act, to_fp16(x) @ w16.t() + b)[0] * dy).sum())

    dz = dy * act_grad(act, z)[1]
    for loss, at, grad, ungated in ((loss_x, x, to_fp16(dz) @ w16, dy @ w), (loss_b, bias, dz.sum(0), dy.sum(0))):
        along = directions(grad, ungated, at)
        assert max(along_errors(loss, at, grad, along)) <= DIFFERENCE
        for name, bad in wrong(grad, ungated).items():
            if name != "ungated" or act != 2:
                assert max(along_errors(loss, at, bad, along)) > 5 * DIFFERENCE, name
