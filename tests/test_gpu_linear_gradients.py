"""dx and dbias of the product's backward pass against differences of its forward pass, along directions in which they are large.

Tolerance: 2 % of the derivative.  Along such a direction (24 rows, K = 256) it is about 16 times what the products' own roundings of 3e-4 of
a row come to, over a step of 2^-8 of x on either side 4e-3; the step's square times a third derivative of the size of the first 3e-3;
dx's roundings 3e-4.  (Measured on formulas in 64 bits with x and weights rounded to fp16: up to 3e-3; every wrong gradient
misses by 10 % and more, test_linear_checks.)"""
import pytest
import torch

import oracle as O
from linear_checks import DIFFERENCE, along_errors, directions, off_the_kink, wrong
from linear_ref import act_grad
from test_gpu_linear import Case

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("fmt", [O.Q4_0, O.Q8_0, O.Q4_K, O.Q6_K])
def test_along_the_gradient(dev, fmt, act):
    import gq
    m, n, k = 24, 96, 256
    c = Case(dev, fmt, m, n, k, seed=18, dtype=torch.float32)
    bias = c.bias.float()
    s = c.x.double() @ c.w.t().contiguous() + bias.double()
    dy = off_the_kink(act, s, c.dy.double()).float()

    def loss(x, b):
        y = gq.linear(fmt, c.packed, x.float(), n, k, bias=b.float(), act=act, resid=c.resid)
        return float((y.double() * dy.double()).sum())

    z = gq.linear(fmt, c.packed, c.x, n, k, bias=bias, act=act, save=True)[1]
    out = gq.linear_bwd(fmt, c.packed, dy, z, n, k, act=act, want_dbias=True)
    dz = dy.double() * act_grad(act, s)[1]  # (the directions are the formula's)
    for name, at, g, flat, fixed in (("dx", c.x, dz @ c.w, dy.double() @ c.w, lambda v: loss(v, bias)),
                                     ("dbias", bias, dz.sum(0), dy.double().sum(0), lambda v: loss(c.x, v))):
        along = directions(g, flat, at)
        errors = along_errors(fixed, at, out[name], along)
        assert max(errors) <= DIFFERENCE, (name, errors)
        for kind, bad in wrong(out[name], flat).items():
            if kind != "ungated" or act != gq.ACT_NONE:
                assert max(along_errors(fixed, at, bad, along)) > DIFFERENCE, (name, kind)
