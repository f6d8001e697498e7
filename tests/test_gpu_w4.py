"""Products with 4-bit weights that have group scales and zero points, against the formula in 64 bits.

Tolerances.  Codes, zero points, scales and x enter exactly; sums are fp32.  A partial sum holds codes with an offset
of up to 128, which is at most 30 times the size of the sum without it (codes spread by 4.6 about their zero
point), and a group's sum takes about 8 roundings of 2^-24: sqrt(8) * 30 * 2^-24 = 5e-6 of the result's norm, 1e-5 with the sums
over groups.  A rounding of the output adds finfo.eps / 2.  A single value is off by at most ten times its row's
rms share of that, beside its rounding."""
import pytest
import torch

from test_ffn_w4_args import act_grad

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
SUM = 1e-5


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def make(dev, n, k, group, seed, scales=torch.float16, zeros=True):
    """(packed, the weights in 64 bits)"""
    import gq
    gen = torch.Generator().manual_seed(seed)
    ng = -(-k // group)
    q = torch.randint(0, 256, (n, -(-k // 2)), generator=gen, dtype=torch.uint8)
    s = ((0.004 + 0.004 * torch.rand(n, ng, generator=gen)) * (1 - 2 * torch.randint(0, 2, (n, ng), generator=gen))).to(scales)
    z = torch.randint(0, 17, (n, ng), generator=gen, dtype=torch.uint8) if zeros else None
    codes = torch.stack([q & 15, q >> 4], 2).reshape(n, -1)[:, :k].double()
    zz = z.double() if zeros else torch.full((n, ng), 8.0, dtype=torch.float64)
    e = torch.arange(k) // group
    w = (s.double()[:, e] * (codes - zz[:, e])).to(dev)
    return gq.w4_pack(q.to(dev), s.to(dev), z.to(dev) if zeros else None, n, k, group), w


def make_x(dev, m, k, dtype, seed):
    return torch.randn(m, k, generator=torch.Generator().manual_seed(1000 + seed)).to(dtype).to(dev)


def check(y, ref, extra=1.0):
    err, t = (y.double() - ref).abs(), half_step(y.dtype)
    rms = ref.pow(2).mean(1, keepdim=True).sqrt()
    assert float(err.norm() / ref.norm()) <= t + SUM * extra
    assert bool((err <= t * ref.abs() + 10 * SUM * extra * rms).all())


SHAPES = [(1, 16, 128), (1, 1, 1), (1, 17, 31), (2, 5, 130), (3, 64, 256), (4, 100, 4096), (5, 33, 1000), (8, 130, 2048), (11, 257, 4090),
          (15, 48, 777), (16, 1000, 512), (16, 16, 14336), (1, 4097, 4096), (1, 300, 14336), (2, 2000, 129)]


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_gemv(dev, group, dtype, m, n, k):
    import gq
    print(f"m={m} n={n} k={k} group={group} {dtype}", flush=True)
    p, w = make(dev, n, k, group, seed=n, scales=torch.bfloat16 if n % 2 else torch.float16, zeros=k % 4 != 0 or n % 2 == 0)
    x = make_x(dev, m, k, dtype, n)
    y = gq.w4_gemv(p, group, x, n, k)
    assert y.dtype == dtype
    check(y, x.double() @ w.t().contiguous())


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", SHAPES[:-2])
def test_gate_up(dev, group, dtype, m, n, k):
    import gq
    print(f"m={m} n={n} k={k} group={group} {dtype}", flush=True)
    (pg, wg), (pu, wu) = make(dev, n, k, group, seed=n), make(dev, n, k, group, seed=n + 1)
    x = make_x(dev, m, k, dtype, n)
    x = (x.double() * 20 / k ** 0.5).to(dtype)  # products of size 1 or so
    for act in (0, 1):
        h = gq.w4_gate_up(pg, pu, group, x, n, k, act=act)
        g, u = x.double() @ wg.t().contiguous(), x.double() @ wu.t().contiguous()
        # (errors of g and of u, each a share of a row's rms, times the other factor: below 4 times its own size)
        check(h, act_grad(act, g)[0] * u, extra=8.0)


# matrices of so many rows that workgroups take four tiles, on four waves and on eight; K with and without a tail
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(3, 22500, 130), (7, 9700, 300), (16, 16401, 256), (12, 9650, 8200), (5, 17000, 129)])
def test_wide(dev, group, dtype, m, n, k):
    import gq
    print(f"m={m} n={n} k={k} group={group} {dtype}", flush=True)
    p, w = make(dev, n, k, group, seed=n)
    x = make_x(dev, m, k, dtype, n)
    check(gq.w4_gemv(p, group, x, n, k), x.double() @ w.t().contiguous())
    if k < 1000:
        h = gq.w4_gate_up(p, p, group, (x.double() / k ** 0.5 * 20).to(dtype), n, k)
        g = (x.double() / k ** 0.5 * 20).to(dtype).double() @ w.t().contiguous()
        check(h, act_grad(0, g)[0] * g, extra=8.0)


@pytest.mark.parametrize("xdt", DTYPES)
@pytest.mark.parametrize("ydt", DTYPES)
@pytest.mark.parametrize("m", [1, 6, 16])
def test_types(dev, xdt, ydt, m):
    import gq
    n, k, group = 200, 640, 64
    (p, w), (p2, w2) = make(dev, n, k, group, seed=1), make(dev, n, k, group, seed=2)
    x = make_x(dev, m, k, xdt, 5)
    y = gq.w4_gemv(p, group, x, n, k, out_dtype=ydt)
    assert y.dtype == ydt
    check(y, x.double() @ w.t().contiguous())
    h = gq.w4_gate_up(p, p2, group, x, n, k, out_dtype=ydt)
    g = x.double() @ w.t().contiguous()
    check(h, act_grad(0, g)[0] * (x.double() @ w2.t().contiguous()), extra=8.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [1, 4, 5, 16])
@pytest.mark.parametrize("at", [0, 1, 3])
def test_nothing_behind_the_outputs(dev, dtype, m, at):
    """Outputs at any alignment, nothing written around them; x at any alignment, with NaN on both sides of it."""
    import gq
    n, k, group = 83, 333, 32
    (p, w), (p2, w2) = make(dev, n, k, group, seed=3), make(dev, n, k, group, seed=4)
    xb = torch.full((at + m * k + 600,), float("nan"), dtype=dtype, device=dev)
    x = xb[at:at + m * k].view(m, k).copy_(make_x(dev, m, k, dtype, 7))
    for call, ref in ((lambda o: gq.w4_gemv(p, group, x, n, k, y=o), x.double() @ w.t().contiguous()),
                      (lambda o: gq.w4_gate_up(p, p2, group, x, n, k, h=o),
                       act_grad(0, x.double() @ w.t().contiguous())[0] * (x.double() @ w2.t().contiguous()))):
        buf = torch.full((at + m * n + 600,), 7.0, dtype=dtype, device=dev)
        out = buf[at:at + m * n].view(m, n)
        call(out)
        check(out, ref, extra=8.0)
        assert bool((buf[:at] == 7).all()) and bool((buf[at + m * n:] == 7).all())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_nonfinite_rows(dev, dtype, bad):
    """A row with an Inf or NaN comes out non-finite, NaN for NaN; the others are as without it."""
    import gq
    m, n, k, group = 5, 64, 512, 128
    p, _ = make(dev, n, k, group, seed=5)
    x = make_x(dev, m, k, dtype, 9)
    ref = gq.w4_gemv(p, group, x, n, k)
    x[2, 200] = bad
    y = gq.w4_gemv(p, group, x, n, k)
    assert not bool(y[2].isfinite().any())
    if bad != bad:
        assert bool(y[2].isnan().all())
    keep = [0, 1, 3, 4]
    assert torch.equal(y[keep], ref[keep])


@pytest.mark.parametrize("dtype,sizes", [(torch.bfloat16, (-90, 90)), (torch.float32, (-90, 90)), (torch.float16, (-8, 3))])
def test_sizes_of_rows(dev, dtype, sizes):
    import gq
    m, n, k, group = 16, 96, 1024, 64
    p, w = make(dev, n, k, group, seed=6)
    s = torch.exp2(torch.randint(*sizes, (m, 1), generator=torch.Generator().manual_seed(3)).double()).to(dev)
    x = (make_x(dev, m, k, dtype, 11).double() * s).to(dtype)
    y = gq.w4_gemv(p, group, x, n, k, out_dtype=torch.float32)
    ref = x.double() @ w.t().contiguous()
    assert float(((y.double() - ref).norm(dim=1) / ref.norm(dim=1)).max()) <= SUM + half_step(torch.float32)


def test_zero_scales_and_equal_codes(dev):
    """Groups that are all zero, and a code that is its zero point everywhere: exact zeros."""
    import gq
    n, k, group = 48, 256, 64
    q = torch.full((n, k // 2), 0x99, dtype=torch.uint8, device=dev)
    z = torch.full((n, k // group), 9, dtype=torch.uint8, device=dev)
    s = torch.ones(n, k // group, dtype=torch.float16, device=dev)
    x = torch.ones(2, k, dtype=torch.bfloat16, device=dev)
    assert bool((gq.w4_gemv(gq.w4_pack(q, s, z, n, k, group), group, x, n, k) == 0).all())
    s.zero_()
    z.zero_()
    assert bool((gq.w4_gemv(gq.w4_pack(q, s, z, n, k, group), group, x, n, k) == 0).all())


def test_captured_and_on_streams(dev):
    import gq
    n, k, group = 1500, 2048, 128
    (p, _), (p2, _) = make(dev, n, k, group, seed=7), make(dev, n, k, group, seed=8)
    for m, dtype in ((1, torch.bfloat16), (9, torch.float32), (16, torch.float16)):
        x = make_x(dev, m, k, dtype, 13)
        y, h = torch.empty(m, n, dtype=dtype, device=dev), torch.empty(m, n, dtype=dtype, device=dev)

        def step():
            gq.w4_gemv(p, group, x, n, k, y=y)
            gq.w4_gate_up(p, p2, group, x, n, k, h=h)

        step()
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        side = torch.cuda.Stream()
        for i in range(3):
            x.copy_(make_x(dev, m, k, dtype, 20 + i))
            y.fill_(float("nan"))
            graph.replay()
            torch.cuda.synchronize()
            got = y.clone(), h.clone()
            with torch.cuda.stream(side):
                other = gq.w4_gemv(p, group, x, n, k), gq.w4_gate_up(p, p2, group, x, n, k)
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(got, other))


def test_binding_refuses(dev):
    import gq
    n, k, group = 64, 256, 64
    p, _ = make(dev, n, k, group, seed=9)
    x = make_x(dev, 2, k, torch.bfloat16, 1)
    for call in (lambda: gq.w4_gemv(p, group, x[:, ::2], n, k // 2), lambda: gq.w4_gemv(p, group, x.t(), n, 2),
                 lambda: gq.w4_gemv(p[:-1], group, x, n, k), lambda: gq.w4_gemv(p, group, x.double(), n, k),
                 lambda: gq.w4_gemv(p, 48, x, n, k), lambda: gq.w4_gemv(p, group, x.repeat(9, 1), n, k),
                 lambda: gq.w4_gemv(p, group, x, n, k, y=torch.empty(2, n + 1, device=dev)),
                 lambda: gq.w4_gate_up(p, p, group, x, n, k, act=2)):
        with pytest.raises(gq.GQError):
            call()
