"""The experts' products held to the figures that their documentation gives, for few tokens and more (figures): g and u of an expert
carry their products' share into h as u act'(g) dg + act(g) du, h is rounded to fp16, and W_down adds its own share.  The errors of one expert's
h are independent of each other: W_down takes them to the root of the sum of its squared weights, which in a column's mean is within a quarter."""
import pytest
import torch

import figures
import oracle as O
from linear_ref import act_grad
from test_gpu_moe import DTYPES, Layer

pytestmark = pytest.mark.gpu


def few(fmt, down, m, top, n, k):
    """Tokens whose rows of x, and of h, are few enough to enter as they are."""
    return m <= 4 and m * figures.padded(fmt, k) <= 64000 and m * top * figures.padded(down, n) <= 66000


def bound(la, x, ids, w, act, shares):
    """y in 64 bits and the error that a row may have, from the shares of gate and up, of h's rounding, and of down."""
    first, half, last = shares
    y, err = torch.zeros_like(x, dtype=torch.float64), torch.zeros(len(x), dtype=torch.float64, device=x.device)
    for j in range(ids.shape[1]):
        for i in range(len(x)):
            gate, up, dn = (t[ids[i, j]] for t in la.w)
            v = figures.taken(x[i:i + 1])
            g, u = v @ gate.t().contiguous(), v @ up.t().contiguous()
            f, d = act_grad(act, g)
            h = f * u
            dg, du = first * (v.pow(2) @ gate.pow(2).t().contiguous()).sqrt(), first * (v.pow(2) @ up.pow(2).t().contiguous()).sqrt()
            dh2 = (u * d * dg).pow(2) + (f * du).pow(2) + (half * h).pow(2)
            out = (dh2 @ dn.pow(2).t().contiguous()).sum().sqrt() * figures.SPREAD + last * figures.terms(h, dn)[0]
            y[i] += w[i, j].double() * (h @ dn.t().contiguous())[0]
            err[i] += w[i, j].double().abs() * out
    return y, err + 2 ** -24 * y.norm(dim=1)


# one to four tokens that fit, tokens of 14336 whose h does not, of long x that does not, more
@pytest.mark.parametrize("fmt,down", [(O.Q4_0, O.Q8_0), (O.Q8_0, O.Q4_K), (O.Q4_K, O.Q6_K), (O.Q6_K, O.Q4_0)])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,e,top,n,k", [(1, 8, 4, 256, 512), (1, 3, 2, 14336, 256), (2, 3, 2, 14336, 256), (3, 3, 2, 14336, 256), (4, 3, 2, 8192, 512),
                                         (4, 3, 2, 256, 15872), (4, 3, 2, 256, 16384), (5, 4, 2, 512, 512), (24, 4, 3, 256, 512)])
def test_products_of_experts(dev, fmt, down, dtype, m, e, top, n, k):
    import gq
    la = Layer(dev, fmt, down, e, n, k, seed=m + top)
    x = la.x(m, dtype)
    gen = torch.Generator().manual_seed(n)
    ids = torch.stack([torch.randperm(e, generator=gen)[:top] for _ in range(m)]).int().to(dev)
    w = (0.1 + torch.rand(m, top, generator=gen)).to(dev)
    y = gq.moe_ffn(fmt, *la.packed[:2], down, la.packed[2], x, ids, w, n, k, e, out_dtype=torch.float32)
    half = figures.SPREAD * figures.HALF
    if few(fmt, down, m, top, n, k):
        shares = figures.few(fmt, dtype), half, figures.few(down, torch.float16)
    else:
        shares = figures.rows(fmt), half, figures.rows(down)
    ref, err = bound(la, x, ids.long(), w, 0, shares)
    diff = (y.double() - ref).norm(dim=1)
    print(f"share {float((diff / err).max()):.3f}")
    assert bool((diff <= err).all()), (diff / err).tolist()


@pytest.mark.parametrize("fmt,down", [(O.Q4_0, O.Q8_0), (O.Q8_0, O.Q4_K), (O.Q4_K, O.Q6_K), (O.Q6_K, O.Q4_0)])
def test_the_same_again(dev, fmt, down):
    """Two calls on the same tokens give the same bits, choice and output, whatever the workspace held."""
    import gq
    la = Layer(dev, fmt, down, 24, 512, 2048, seed=2)
    la.router *= 1 / la.size
    for m in (1, 3, 4, 5, 16, 17, 37, 64):
        x, ws = la.x(m, torch.bfloat16), gq.Workspace(dev)

        def call():
            return gq.moe_layer(fmt, *la.packed[:2], down, la.packed[2], la.router, x, la.n, la.k, la.e, 6, save=True, workspace=ws)

        first = [t.clone() for t in call()]
        for _ in range(3):
            ws.ensure(1).fill_(0xFF)
            assert all(torch.equal(a, b) for a, b in zip(first, call()))
