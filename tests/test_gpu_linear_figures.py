"""The product with its epilogue held to the figures that its documentation gives, path by path.

Tolerances.  An activation z s(p): the sigmoid's argument is off by five and a half half steps of fp32, 3.3e-7 |p| of s, its exponential,
reciprocal and products by six, 3.6e-7; results below fp32's range are flushed, 1e-30.  Products: figures."""
import math

import pytest
import torch

import figures
import oracle as O
from linear_ref import act_grad
from test_gpu_linear import DTYPES, Case

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


# rows that are few and fit LDS together, the last that do and the first that do not, up to 16, tiles
@pytest.mark.parametrize("fmt", [O.Q4_0, O.Q8_0, O.Q4_K, O.Q6_K])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 512), (1, 14336), (1, 65536), (1, 65792), (2, 4096), (2, 32768), (3, 21760), (3, 22016), (4, 1024), (4, 16384), (4, 16640),
                                 (4, 20480), (5, 512), (11, 4096), (16, 14336), (17, 1024), (60, 4096), (200, 2048)])
def test_products(dev, fmt, dtype, m, k):
    import gq
    n = 160
    c = Case(dev, fmt, m, n, k, seed=k % 7, dtype=dtype, bias=False, resid=False)
    y = gq.linear(fmt, c.packed, c.x, n, k, out_dtype=torch.float32)
    err = (y.double() - figures.taken(c.x) @ c.w.t().contiguous()).norm(dim=1) / figures.terms(c.x, c.w)
    print(f"share {float(err.max()):.3e} of {figures.linear(fmt, m, k, dtype):.3e}")
    assert float(err.max()) <= figures.linear(fmt, m, k, dtype), float(err.max())


@pytest.mark.parametrize("fmt", [O.Q4_0, O.Q8_0, O.Q4_K, O.Q6_K])
@pytest.mark.parametrize("m,n,k", [(1, 256, 512), (8, 1000, 1024), (70, 513, 512), (300, 2048, 512)])
def test_input_gradients(dev, fmt, m, n, k):
    """dx: dz to fp16 and the weights as in the tiles."""
    import gq
    c = Case(dev, fmt, m, n, k, seed=n % 7, dtype=torch.float16)
    dx = gq.linear_bwd(fmt, c.packed, c.dy, None, n, k, dx_dtype=torch.float32, want_dz=False)["dx"]
    rows = c.dy.double().norm(dim=1) > 0
    err = (dx.double() - figures.taken(c.dy.float()) @ c.w).norm(dim=1)[rows] / figures.terms(c.dy, c.w.t())[rows]
    print(f"share {float(err.max()):.3e} of {figures.tiles(fmt):.3e}")
    assert float(err.max()) <= figures.tiles(fmt), float(err.max())


@pytest.mark.parametrize("fmt", [O.Q4_0, O.Q8_0, O.Q4_K, O.Q6_K])
@pytest.mark.parametrize("m,k", [(1, 512), (4, 4096), (5, 512), (16, 4096), (40, 512), (300, 1024)])
def test_subnormal_fp16_rows(dev, fmt, m, k):
    """fp16 rows of subnormals alone, and of subnormals beside a 1 (2^14 x / 16, the 4-bit formats' smallest, is still normal), on the paths
    that convert x and on those that take it as it is: no value is flushed."""
    import gq
    n = 160
    c = Case(dev, fmt, m, n, k, seed=3, dtype=torch.float32, bias=False, resid=False)
    x = c.x.double() / c.x.double().abs().max() * 2.0 ** -15
    c.x = x.to(torch.float16)
    assert float(c.x.abs().max()) < 2.0 ** -14 and int((c.x != 0).sum()) > 0.9 * c.x.numel()
    for large in (False, True):
        if large:
            c.x[:, 3] = 1.0
        y = gq.linear(fmt, c.packed, c.x, n, k, out_dtype=torch.float32)
        ref = c.x.double() @ c.w.t().contiguous()
        err = (y.double() - ref).norm(dim=1)
        assert bool((err <= figures.linear(fmt, m, k, torch.float16) * figures.terms(c.x, c.w)).all())
        if not large:
            assert bool((ref.norm(dim=1) > 0).all())


@pytest.mark.parametrize("fmt", [O.Q4_0, O.Q8_0, O.Q4_K, O.Q6_K])
def test_the_same_again(dev, fmt):
    """Two calls on the same inputs give the same bits, on every path and for every output."""
    import gq
    n, k = 1030, 4096
    for m in (1, 3, 4, 9, 16, 40, 203, 509):
        c = Case(dev, fmt, m, n, k, seed=m, dtype=torch.float16)
        ws = gq.Workspace(dev)

        def call():
            y, z = gq.linear(fmt, c.packed, c.x, n, k, bias=c.bias, act=1, resid=c.resid, save=True, workspace=ws)
            return y, z, *gq.linear_bwd(fmt, c.packed, c.dy, c.z, n, k, act=1, want_dbias=True, workspace=ws).values()

        first = [t.clone() for t in call()]
        for _ in range(3):
            ws.ensure(1).fill_(0xFF)  # (what a workspace held before is of no account)
            assert all(torch.equal(a, b) for a, b in zip(first, call()))


@pytest.mark.parametrize("dtype", DTYPES)
def test_bias_gradient_over_blocks_of_rows(dev, dtype):
    """More rows than a block of the bias gradient without dx takes (2^20): its last block is of fewer rows than workgroups share."""
    import gq
    m, n, k = (1 << 20) + 100, 9, 32
    gen = torch.Generator(device=dev).manual_seed(4)
    dy, z = (torch.randn(m, n, generator=gen, device=dev).to(dtype) for _ in range(2))
    w = gq.repack(O.Q8_0, torch.zeros(gq.gguf_bytes(O.Q8_0, n, k), dtype=torch.uint8, device=dev), n, k)
    out = gq.linear_bwd(O.Q8_0, w, dy, z, n, k, act=3, want_dx=False, want_dbias=True)
    dz = dy.double() * (z.double() > 0)
    assert torch.equal(out["dz"].double(), dz)
    # (a workgroup adds its 4097 rows in fp32: as many sums that grow as a root, each off by up to half a step; 256 of them are added in 64 bits)
    err = (out["dbias"].double() - dz.sum(0)).abs()
    assert bool((err <= 2 ** -24 * 4097 ** 0.5 * 4 * dz.pow(2).sum(0).sqrt() + 2 ** -24 * dz.sum(0).abs()).all())


@pytest.mark.parametrize("fmt", [O.Q4_0, O.Q8_0, O.Q4_K, O.Q6_K])
@pytest.mark.parametrize("n", [1, 3])
def test_longest_rows(dev, fmt, n):
    """K = 2^24, the largest: one row, sixteen, and more in blocks of sixteen; its gradient.  (fp32 sums of 2^17 units of 128 terms, one after the
    other in four waves: 2^-24 256 of them beside the shares.)"""
    import gq
    k, m = 1 << 24, 17
    b = O.gen_weights(fmt, n, k, seed=n)
    w, packed = torch.from_numpy(O.dequant(fmt, b).reshape(n, k)).to(dev), gq.repack(fmt, torch.from_numpy(b).to(dev), n, k)
    gen = torch.Generator(device=dev).manual_seed(1)
    x = torch.randn(m, k, generator=gen, device=dev).to(torch.float16)
    ws = gq.Workspace(dev, gq.linear_workspace_bytes(fmt, m, n, k))
    ref = torch.stack([(w.double() * r.double()).sum(1) for r in x])
    size = torch.stack([(w.double() * r.double()).pow(2).sum(1).sqrt() for r in x])
    for rows in (1, 16, 17):
        y = gq.linear(fmt, packed, x[:rows], n, k, out_dtype=torch.float32, workspace=ws)
        share = 4 * (figures.tiles(fmt) if rows > 16 else figures.rows(fmt)) + 2 ** -16  # (single sums: within four of their deviations)
        assert bool(((y.double() - ref[:rows]).abs() <= share * size[:rows]).all())
    dy = torch.randn(3, n, generator=gen, device=dev)
    dx = gq.linear_bwd(fmt, packed, dy, None, n, k, want_dz=False, workspace=gq.Workspace(dev))["dx"]
    dz = figures.taken(dy).float()
    for r in range(3):
        # (a row's norm, as everywhere: a single weight of Q4_K whose minimum cancels it is 0 with an error of the minimum's half step)
        want, size = (dz[r, :, None] * w).double().sum(0), (dz[r, :, None] * w).double().norm()
        assert float((dx[r].double() - want).norm()) <= figures.tiles(fmt) * float(size)
