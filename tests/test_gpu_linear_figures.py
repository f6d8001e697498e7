"""The product with its epilogue held to the figures that its documentation gives, path by path.

Tolerances.  An activation z s(p): the sigmoid's argument is off by five and a half half steps of fp32, 3.3e-7 |p| of s, its exponential,
reciprocal and products by six, 3.6e-7; results below fp32's range are flushed, 1e-30."""
import math

import pytest
import torch

import oracle as O
from linear_ref import act_grad

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", [0, 1])
@pytest.mark.parametrize("m", [1, 8, 40])
def test_both_sides_of_an_activation(dev, act, m):
    """Sums of zero weights (the bias alone) over the whole range: where the sigmoid is 0 the output is, to the last digits, not a
    share of the sum, and the derivative too."""
    import gq
    k = 64
    at = torch.cat([torch.linspace(-110, 110, 1761), torch.tensor([-3e38, -1e30, -1e20, -1e10, -1e5, -1e3, 1e3, 1e10, 1e30, 1e-30, -1e-30, 0.0])])
    z = at.float().to(dev)
    n = z.shape[0]
    packed = gq.repack(O.Q4_0, torch.zeros(n * k // 32 * 18, dtype=torch.uint8, device=dev), n, k)
    x, one = torch.ones(m, k, device=dev), torch.ones(m, n, device=dev)
    y, kept = gq.linear(O.Q4_0, packed, x, n, k, bias=z, act=act, save=True)
    assert torch.equal(kept, z.repeat(m, 1))
    dz = gq.linear_bwd(O.Q4_0, packed, one, kept, n, k, act=act, want_dx=False)["dz"]
    t = z.double().clamp(-1e4, 1e4)  # (beyond: 0, 1, and z)
    f, d = act_grad(act, t)
    f = torch.where(z > 1e4, z.double(), f)
    b = 2 * math.sqrt(2 / math.pi)
    p, dp = (t, torch.ones_like(t)) if act == 0 else (b * (t + 0.044715 * t ** 3), b * (1 + 3 * 0.044715 * t ** 2))
    s = torch.sigmoid(p)
    rel = 4e-7 * p.abs().clamp(max=100) + 1e-6
    assert bool(((y.double() - f).abs() <= rel * f.abs() + 1e-30).all())
    assert bool(((dz.double() - d).abs() <= rel * (s + (t * dp).abs() * s * torch.sigmoid(-p)) + 2 ** -24 * (t * dp).abs() * s + 1e-30).all())
