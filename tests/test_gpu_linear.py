"""The product with bias, activation and residual over T16 weights and its backward pass against the formulas in 64 bits.

Tolerances.  A product over K is a sum of independent terms, so its error, as a share of a row's norm, is that of one
term: x to fp16 (2^-11 at most, after a power-of-two scale) and the weight to fp16 (2^-11; the k-quants with a minimum round
twice, and there to 2^-11 of a product up to three times the weight's size) -- under 1e-3, the bound of every product of this
library.  Proof of what the share is of: with term errors t_k e_k, |e_k| <= e and independent signs, the sum's error is e times the
root of the sum of t_k^2, whatever the sum itself is; a row of x that is nearly orthogonal to the columns' common part (weights
with minima have one) has products smaller than that.  So dz is 1e-3 of the root mean square over the columns of sqrt(sum_k
(x_k w_k)^2), the same size along a row, and y = act(z) + resid takes it as act'(z) dz.  A rounding of the output adds finfo.eps / 2.  Elementwise gradients are fp32
arithmetic: ten roundings of 2^-24 and a 2^-21 exponential.  A sum of M terms in fp32 over workgroups of M / 256 rows, then in
64 bits: (M / 256 + 2) 2^-24 of the sum of magnitudes."""
import pytest
import torch

import oracle as O
from linear_ref import act_grad

pytestmark = pytest.mark.gpu
FMTS = [O.Q4_0, O.Q8_0, O.Q4_K, O.Q4_K_GGML, O.Q6_K, O.Q6_K_GGML]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
PRODUCT = 1e-3


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def weights(dev, fmt, n, k, seed):
    import gq
    b = O.gen_weights(fmt, n, k, seed=seed)
    return gq.repack(fmt, torch.from_numpy(b).to(dev), n, k), torch.from_numpy(O.dequant(fmt, b).reshape(n, k)).to(dev).double()


class Case:
    def __init__(self, dev, fmt, m, n, k, seed=0, dtype=torch.bfloat16, bias=True, resid=True):
        print(f"fmt={fmt} m={m} n={n} k={k} dtype={dtype} seed={seed}", flush=True)
        self.fmt, self.m, self.n, self.k = fmt, m, n, k
        self.packed, self.w = weights(dev, fmt, n, k, 9000 + seed)
        size = float(self.w.pow(2).mean().sqrt()) * k ** 0.5  # products of size 1.5
        gen = torch.Generator().manual_seed(seed)
        self.x = (torch.randn(m, k, generator=gen) * 1.5 / size).to(dtype).to(dev)
        self.bias = (0.5 * torch.randn(n, generator=gen)).to(DTYPES[seed % 3]).to(dev) if bias else None
        self.resid = (2 * torch.randn(m, n, generator=gen)).to(dtype).to(dev) if resid else None
        self.z = (1.5 * torch.randn(m, n, generator=gen)).to(dtype).to(dev)
        tok = torch.exp(torch.randn(m, 1, generator=gen)) * (torch.rand(m, 1, generator=gen) > 0.15)
        self.dy = (0.1 * tok * torch.randn(m, n, generator=gen)).to(dtype).to(dev)


def check_forward(c, act, y, z, dtype):
    p = c.x.double() @ c.w.t().contiguous()
    s = p if c.bias is None else p + c.bias.double()
    f, d = act_grad(act, s)
    ref = f if c.resid is None else f + c.resid.double()
    rms = (c.x.double().pow(2) @ c.w.pow(2).t().contiguous()).mean(1).sqrt()
    bound = PRODUCT * rms * d.norm(dim=1) + half_step(dtype) * ref.norm(dim=1)
    # a kink: where an error moves z over 0, relu's difference is below that error
    if act == 3:
        bound = PRODUCT * rms * c.n ** 0.5 + half_step(dtype) * ref.norm(dim=1)
    assert bool(((y.double() - ref).norm(dim=1) <= bound + 1e-30).all())
    if z is not None:
        bound = PRODUCT * rms * c.n ** 0.5 + half_step(dtype) * s.norm(dim=1)
        assert bool(((z.double() - s).norm(dim=1) <= bound + 1e-30).all())


def check_grads(c, act, out, dtype, z=None):
    _, d = act_grad(act, c.z.double())
    dz = c.dy.double() * d
    tiny = float(torch.finfo(dtype).tiny) * float(torch.finfo(dtype).eps)
    size = c.dy.double().abs() * 2  # (act' is at most 1.13)
    if out["dz"] is not None:
        err = (out["dz"].double() - dz).abs()
        assert bool((err <= half_step(dtype) * dz.abs() + 2e-6 * size + tiny).all())
    if out["dbias"] is not None:
        err = (out["dbias"].double() - dz.sum(0)).abs()
        per = 2e-6 * size.sum(0) + (c.m / 256 + 2) * 2 ** -24 * dz.abs().sum(0)
        assert bool((err <= per).all())
    if out["dx"] is not None:
        dx = dz @ c.w
        diff, norm = (out["dx"].double() - dx).norm(dim=1), dx.norm(dim=1)
        assert bool((diff <= (PRODUCT + half_step(out["dx"].dtype)) * norm).all())


# every format, rows and columns that end inside a tile, one row and one column
SHAPES = [(1, 64, 256), (2, 1, 256), (3, 17, 512), (4, 2050, 256), (5, 100, 256), (16, 48, 1024), (17, 33, 256), (33, 200, 768),
          (64, 129, 512), (65, 64, 1280), (130, 500, 256), (257, 300, 512), (520, 130, 256)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_forward(dev, fmt, m, n, k):
    import gq
    dtype, act = DTYPES[(m + n) % 3], (m + fmt) % 4
    c = Case(dev, fmt, m, n, k, seed=m, dtype=dtype)
    y, z = gq.linear(fmt, c.packed, c.x, n, k, bias=c.bias, act=act, resid=c.resid, save=True)
    check_forward(c, act, y, z, dtype)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_backward(dev, fmt, m, n, k):
    import gq
    dtype, act = DTYPES[(m + n + 1) % 3], (m + fmt + 2) % 4
    c = Case(dev, fmt, m, n, k, seed=m, dtype=dtype)
    check_grads(c, act, gq.linear_bwd(fmt, c.packed, c.dy, c.z, n, k, act=act, want_dbias=True), dtype)
