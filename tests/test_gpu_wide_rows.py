"""Finite rows near the ends of fp32's range: x, and an expert's h, go to fp16 under a power of two whatever their size, so their
products keep the precision of ordinary rows (those of one to four bf16 rows, which enter as they are, are bounded: test_gpu_large_values).

Tolerance: PRODUCT of test_gpu_linear, of the root of a row's sum of squared terms; outputs are fp32, far from its subnormals."""
import pytest
import torch

import oracle as O
from test_gpu_linear import PRODUCT, Case

pytestmark = pytest.mark.gpu
FMTS = [O.Q4_0, O.Q8_0, O.Q4_K, O.Q6_K]


def wide(dev, fmt, m, n, k, dtype):
    """A case whose rows are up to 2^115 .. 2^125 and 2^-109 .. 2^-117 in turn, an ordinary one and one of zeros behind."""
    c = Case(dev, fmt, m, n, k, seed=m + 1, dtype=dtype, bias=False, resid=False)
    s = torch.tensor([2.0 ** (122 if i % 2 == 0 else -112) for i in range(m)], dtype=torch.float64, device=dev)
    if m > 3:
        s[-2], s[-1] = 1, 0
    c.x = (c.x.double() * s[:, None]).to(dtype)
    assert bool(c.x.isfinite().all()) and float(c.x[0].abs().max()) > 2.0 ** 115
    return c


def close(c, y):
    p = c.x.double() @ c.w.t().contiguous()
    rms = (c.x.double().pow(2) @ c.w.pow(2).t().contiguous()).mean(1).sqrt()
    err = (y.double() - p).norm(dim=1)
    assert bool((err <= PRODUCT * rms * c.n ** 0.5).all()), (err / (rms * c.n ** 0.5)).tolist()


# (1 to 4 fp32 rows, 5 to 16, tiles; fp32 rows longer than a workgroup keeps in registers; 1024 rows and more are converted a wave a row)
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,k,dtype", [(1, 512, torch.float32), (4, 512, torch.float32), (5, 512, torch.bfloat16), (16, 4608, torch.float32),
                                       (40, 512, torch.bfloat16), (40, 512, torch.float32), (20, 33024, torch.float32), (1100, 512, torch.float32)])
def test_linear(dev, fmt, m, k, dtype):
    import gq
    n = 100
    c = wide(dev, fmt, m, n, k, dtype)
    close(c, gq.linear(fmt, c.packed, c.x, n, k, out_dtype=torch.float32))


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,k,dtype", [(1, 512, torch.float32), (4, 4608, torch.float32), (16, 512, torch.bfloat16), (40, 512, torch.float32), (300, 512, torch.bfloat16)])
def test_front(dev, fmt, m, k, dtype):
    import gq
    n = 100
    c = wide(dev, fmt, m, n, k, dtype)
    _, g, u = gq.ffn_gate_up(fmt, c.packed, c.packed, c.x, n, k, save=True, out_dtype=torch.float32)
    close(c, g)
    assert torch.equal(g, u)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,k", [(40, 512), (200, 512), (300, 4608), (1100, 512)])
def test_gemm(dev, fmt, m, k):
    import gq
    n = 272
    c = wide(dev, fmt, m, n, k, torch.float32)
    close(c, gq.matmul(fmt, c.packed, c.x, n, k))
    if fmt == O.Q6_K and k > 4096:  # (gq_matmul's alone)
        return
    for dtype in (torch.float32, torch.bfloat16):
        c = wide(dev, fmt, m, n, k, dtype)
        close(c, gq.gemm(fmt, c.packed, c.x, n, k, workspace=gq.Workspace(dev)))


def test_windows_of_one_row(dev):
    """Q6_K of more than 4096 columns scales windows of 256 apart: one of up to 2^118 beside ordinary and tiny ones."""
    import gq
    m, n, k = 200, 272, 4608
    c = wide(dev, O.Q6_K, m, n, k, torch.float32)
    c.x[0] = 2.0 ** -70 * c.x[0]
    c.x[0, 300] = 2.0 ** 118
    c.x[2, 512:] = 0
    close(c, gq.matmul(O.Q6_K, c.packed, c.x, n, k))


# (1, 2 to 8, 9 to 16 rows; K short, of several parts, and more than a workgroup stages at once)
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", [1, 2, 8, 13, 16])
@pytest.mark.parametrize("n,k", [(100, 512), (4096, 4608), (272, 14336)])
def test_gemv(dev, fmt, m, n, k):
    import gq
    c = wide(dev, fmt, m, n, k, torch.float32)
    close(c, gq.gemv(fmt, c.packed, c.x, n, k, workspace=gq.Workspace(dev)))
    close(c, gq.matmul(fmt, c.packed, c.x, n, k))
    for y in gq.gemv_multi(fmt, [(c.packed, n), (c.packed, n)], c.x, k) if m <= 4 else ():  # (which takes no more)
        close(c, y)


@pytest.mark.parametrize("m", [1, 2, 8, 16, 40, 200])
@pytest.mark.parametrize("n,k", [(100, 512), (272, 4608)])
def test_fp16_weights(dev, m, n, k):
    import gq
    c = wide(dev, O.Q8_0, m, n, k, torch.float32)
    w = c.w.to(torch.float16)
    c.w = w.double()
    close(c, gq.gemm_f16w(w, c.x, n, k))


@pytest.mark.parametrize("fmt,down", [(O.Q4_0, O.Q8_0), (O.Q8_0, O.Q4_K), (O.Q4_K, O.Q6_K), (O.Q6_K, O.Q4_0)])
@pytest.mark.parametrize("m", [1, 4, 5, 64])
@pytest.mark.parametrize("size", [60, 58, 56])
def test_hidden_values_of_experts(dev, fmt, down, m, size):
    """h = silu(g) u of g and u about 2^size (h to 2^124 and more), and of 2^-58.  Tokens with an h or a sum of its products past 2^126 are
    not looked at: W_down's rows of up to 55 times h's size take them past fp32's largest."""
    import gq
    from test_gpu_moe import Layer
    e, n, k = 3, 256, 256
    la = Layer(dev, fmt, down, e, n, k, seed=m)
    x = la.x(m, torch.float32)
    x[0::2] *= 2.0 ** size
    x[1::2] *= 2.0 ** -58
    gen = torch.Generator().manual_seed(m)
    ids = torch.stack([torch.randperm(e, generator=gen)[:2] for _ in range(m)]).int().to(dev)
    w = (0.25 + torch.rand(m, 2, generator=gen)).to(dev)
    y = gq.moe_ffn(fmt, *la.packed[:2], down, la.packed[2], x, ids, w, n, k, e)
    ref, err = la.reference(x, ids, w, 0, None)
    fits = ref.abs().amax(1) < 2.0 ** 126
    for j in range(2):
        for i in range(m):
            g, u = (la.w[t][ids[i, j]] @ x[i].double() for t in (0, 1))
            h = torch.nn.functional.silu(g) * u
            fits[i] &= bool((h.abs() < 2.0 ** 126).all() and ((la.w[2][ids[i, j]] @ h).abs() < 2.0 ** 126).all())
    diff = (y.double() - ref).norm(dim=1)
    assert bool((diff <= err)[fits].all()), (diff / err)[fits].tolist()
    assert size > 56 or bool(fits.all())


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,dtype", [(1, torch.float32), (4, torch.float32), (5, torch.bfloat16), (20, torch.float32), (64, torch.bfloat16)])
def test_tokens_at_shut_gates(dev, fmt, m, dtype):
    """Tokens of up to 2^120 whose gates' weights are zeros: h = 0, y is the residual, not a NaN, for the layer and its halves alike."""
    import gq
    from test_gpu_moe import Layer
    e, n, k = 4, 256, 256
    la = Layer(dev, fmt, O.Q8_0, e, n, k, seed=m)
    shut = gq.repack(fmt, torch.zeros(gq.gguf_bytes(fmt, e * n, k), dtype=torch.uint8, device=dev), e * n, k)
    # (weights of up to 32, whose sums with x of up to 1 stay below 2^9: u fits fp32)
    x = (la.x(m, torch.float32) * 2.0 ** 118 / la.size).clamp(-2.0 ** 118, 2.0 ** 118).to(dtype)
    assert float((x.double() @ la.w[1].reshape(-1, k).t().contiguous()).abs().max()) < 2.0 ** 127
    resid = torch.randn(m, k, generator=la.gen).to(dtype).to(dev)
    y, ids, w = gq.moe_layer(fmt, shut, la.packed[1], O.Q8_0, la.packed[2], la.router, x, n, k, e, 2, score=1, resid=resid, save=True)
    assert torch.equal(y, resid)
    assert torch.equal(gq.moe_ffn(fmt, shut, la.packed[1], O.Q8_0, la.packed[2], x, ids, w, n, k, e, resid=resid), resid)
