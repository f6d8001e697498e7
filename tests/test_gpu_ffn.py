"""The gated feed-forward front over T16 weights and its backward pass against the formulas in 64 bits.

Tolerances.  A product over K is a sum of independent terms, so its error, as a share of a row's norm, is that of one
term: x to fp16 (2^-11 at most, f32 and bf16 inputs scaled by a power of two first) and the weight to fp16 (2^-11;
the k-quants with a minimum round twice, and there to 2^-11 of a product up to three times the weight's size) -- under 1e-3,
the bound of every product of this library.  Such an error has one size along a row, whatever the value it falls
on, so in h = act(g) u it counts as dh = u act'(g) dg + act(g) du with dg, du of 1e-3 of the rms of their row: a row whose gates
are mostly closed is small itself while u act'(g) dg is not.  A rounding of the output adds finfo.eps / 2.  dg and du are fp32 arithmetic: ten roundings of 2^-24 and a 2^-21 exponential."""
import numpy as np
import pytest
import torch

import oracle as O
from test_ffn_w4_args import act_grad

pytestmark = pytest.mark.gpu
FMTS = [O.Q4_0, O.Q8_0, O.Q4_K, O.Q4_K_GGML, O.Q6_K, O.Q6_K_GGML]
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
PRODUCT = 1e-3


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def worst_row(a, b):
    """The largest error of a row as a share of the row's norm; rows that are zero have to be zero."""
    d, n = (a.double() - b).norm(dim=1), b.norm(dim=1)
    assert bool((d[n == 0] == 0).all())
    return float((d[n > 0] / n[n > 0]).max()) if bool((n > 0).any()) else 0.0


class Case:
    def __init__(self, dev, fmt, m, n, k, seed=0, dtype=torch.bfloat16):
        import gq
        print(f"fmt={fmt} m={m} n={n} k={k} dtype={dtype} seed={seed}", flush=True)
        self.fmt, self.m, self.n, self.k = fmt, m, n, k
        self.packed, self.w = [], []
        for i in range(2):
            b = O.gen_weights(fmt, n, k, seed=7000 + 2 * seed + i)
            self.packed.append(gq.repack(fmt, torch.from_numpy(b).to(dev), n, k))
            self.w.append(torch.from_numpy(O.dequant(fmt, b).reshape(n, k)).to(dev).double())
        size = float(self.w[0].pow(2).mean().sqrt()) * k ** 0.5  # products of size 1.5
        gen = torch.Generator().manual_seed(seed)
        self.x = (torch.randn(m, k, generator=gen) * 1.5 / size).to(dtype).to(dev)
        self.g = (1.5 * torch.randn(m, n, generator=gen)).to(dtype).to(dev)
        self.u = (1.5 * torch.randn(m, n, generator=gen)).to(dtype).to(dev)
        tok = torch.exp(torch.randn(m, 1, generator=gen)) * (torch.rand(m, 1, generator=gen) > 0.15)
        self.dh = (0.1 * tok * torch.randn(m, n, generator=gen)).to(dtype).to(dev)

    def front(self, act):
        x = self.x.double()
        g, u = x @ self.w[0].t().contiguous(), x @ self.w[1].t().contiguous()
        return act_grad(act, g)[0] * u, g, u

    def grads(self, act):
        f, d = act_grad(act, self.g.double())
        dg, du = self.dh.double() * self.u.double() * d, self.dh.double() * f
        return dg @ self.w[0] + du @ self.w[1], dg, du


def check_front(c, act, out, dtype):
    h, g, u = c.front(act)
    f, d = act_grad(act, g)
    rms = [t.pow(2).mean(1).sqrt() for t in (g, u)]
    bound = PRODUCT * (rms[0] * (u * d).norm(dim=1) + rms[1] * f.norm(dim=1)) + half_step(dtype) * h.norm(dim=1)
    assert bool(((out[0].double() - h).norm(dim=1) <= bound + 1e-30).all())
    for o, r in ((out[1], g), (out[2], u)):
        if o is not None:
            assert worst_row(o, r) <= PRODUCT + half_step(dtype)


def check_grads(c, act, out, dtype):
    dx, dg, du = c.grads(act)
    f, _ = act_grad(act, c.g.double())
    tiny = float(torch.finfo(dtype).tiny) * float(torch.finfo(dtype).eps)
    for name, r, size in (("dg", dg, c.dh.double() * c.u.double()), ("du", du, c.dh.double() * c.g.double())):
        if out[name] is not None:
            err = (out[name].double() - r).abs()
            assert bool((err <= half_step(dtype) * r.abs() + 2e-6 * size.abs() + tiny).all()), name
    if out["dx"] is not None:
        assert worst_row(out["dx"], dx) <= PRODUCT + half_step(out["dx"].dtype)


# every format, rows and columns that end inside a tile, one row and one column
SHAPES = [(1, 64, 256), (2, 1, 256), (3, 17, 512), (5, 100, 256), (16, 48, 1024), (17, 33, 256), (33, 200, 768), (64, 129, 512),
          (65, 64, 1280), (130, 500, 256), (257, 300, 512), (520, 130, 256)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_front(dev, fmt, m, n, k):
    import gq
    dtype = DTYPES[(m + n) % 3]
    c = Case(dev, fmt, m, n, k, seed=m, dtype=dtype)
    act = (m + fmt) % 2
    check_front(c, act, gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, act=act, save=True), dtype)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_backward(dev, fmt, m, n, k):
    import gq
    dtype = DTYPES[(m + n + 1) % 3]
    c = Case(dev, fmt, m, n, k, seed=m, dtype=dtype)
    act = (m + fmt) % 2
    check_grads(c, act, gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k, act=act), dtype)


# formats with blocks of 32: K that is no whole chunk of the layout
@pytest.mark.parametrize("fmt", [O.Q4_0, O.Q8_0])
@pytest.mark.parametrize("m,n,k", [(1, 16, 32), (4, 40, 96), (20, 65, 160), (100, 70, 4128), (300, 129, 224)])
def test_short_chunks(dev, fmt, m, n, k):
    import gq
    c = Case(dev, fmt, m, n, k, seed=k, dtype=torch.float16)
    check_front(c, 0, gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, save=True), torch.float16)
    check_grads(c, 0, gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k), torch.float16)


# long rows, many rows, few rows of a wide matrix
@pytest.mark.parametrize("fmt", [O.Q4_0, O.Q8_0, O.Q4_K, O.Q6_K])
@pytest.mark.parametrize("m,n,k", [(1, 4099, 4096), (7, 1030, 8192), (12, 2100, 1024), (16, 14336, 256), (40, 3001, 2048),
                                   (200, 4100, 1024), (700, 1500, 2304), (2050, 520, 512), (1500, 2100, 4096)])
def test_large(dev, fmt, m, n, k):
    import gq
    c = Case(dev, fmt, m, n, k, seed=n, dtype=torch.bfloat16)
    check_front(c, 1, gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, act=1, save=True), torch.bfloat16)
    check_grads(c, 1, gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k, act=1), torch.bfloat16)


@pytest.mark.parametrize("xdt", DTYPES)
@pytest.mark.parametrize("hdt", DTYPES)
@pytest.mark.parametrize("m", [1, 8, 40, 150])
def test_types(dev, xdt, hdt, m):
    import gq
    fmt, n, k = O.Q4_K, 272, 512
    c = Case(dev, fmt, m, n, k, seed=3, dtype=xdt)
    h = gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, out_dtype=hdt)
    assert h.dtype == hdt
    check_front(c, 0, (h, None, None), hdt)
    out = gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k, dx_dtype=hdt)
    assert out["dx"].dtype == hdt and out["dg"].dtype == xdt
    check_grads(c, 0, out, xdt)


@pytest.mark.parametrize("m", [1, 16, 33, 260])
def test_wanted_outputs_alone(dev, m):
    """Each output by itself gives what it gives with the others."""
    import gq
    fmt, n, k = O.Q8_0, 100, 256
    c = Case(dev, fmt, m, n, k, seed=5, dtype=torch.bfloat16)
    h, g, u = gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, save=True)
    assert torch.equal(gq.ffn_gate_up(fmt, *c.packed, c.x, n, k), h)
    only_u = gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, u=torch.empty_like(u))
    assert only_u[1] is None and torch.equal(only_u[0], h) and torch.equal(only_u[2], u)
    full = gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k)
    part = gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k, want_dgu=False)
    assert part["dg"] is None and part["du"] is None and torch.equal(part["dx"], full["dx"])
    part = gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k, want_dx=False)
    assert part["dx"] is None and torch.equal(part["dg"], full["dg"]) and torch.equal(part["du"], full["du"])
    # dg over g, du over dh
    gg, dd = c.g.clone(), c.dh.clone()
    out = gq.ffn_gate_up_bwd(fmt, *c.packed, dd, gg, c.u, n, k, dg=gg, du=dd)
    assert torch.equal(gg, full["dg"]) and torch.equal(dd, full["du"]) and torch.equal(out["dx"], full["dx"])


@pytest.mark.parametrize("m", [1, 5, 16, 20, 64, 100, 300])
@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_behind_the_outputs(dev, m, dtype):
    """Rows behind the last stay as they were, at any alignment of the operands."""
    import gq
    fmt, n, k = O.Q4_0, 101, 288
    c = Case(dev, fmt, m, n, k, seed=9, dtype=dtype)

    def guarded(rows, cols, at):
        buf = torch.full((at + rows * cols + 2000,), 7.0, dtype=dtype, device=dev)
        return buf, buf[at:at + rows * cols].view(rows, cols)

    for at in (0, 1, 3):
        bufs, outs = zip(*[guarded(m, cols, at) for cols in (n, n, n, n, n, k)])
        x = guarded(m, k, at)[1].copy_(c.x)
        dh, g, u = (guarded(m, n, at)[1].copy_(t) for t in (c.dh, c.g, c.u))
        gq.ffn_gate_up(fmt, *c.packed, x, n, k, h=outs[0], g=outs[1], u=outs[2])
        check_front(c, 0, outs[:3], dtype)
        gq.ffn_gate_up_bwd(fmt, *c.packed, dh, g, u, n, k, dg=outs[3], du=outs[4], dx=outs[5])
        check_grads(c, 0, {"dg": outs[3], "du": outs[4], "dx": outs[5]}, dtype)
        for buf, o in zip(bufs, outs):
            assert bool((buf[:at] == 7).all()) and bool((buf[at + o.numel():] == 7).all())


@pytest.mark.parametrize("m", [1, 8, 48, 200])
def test_sizes_of_rows(dev, m):
    """Rows far outside fp16's range, in both directions, keep their precision."""
    import gq
    fmt, n, k = O.Q8_0, 128, 512
    c = Case(dev, fmt, m, n, k, seed=11, dtype=torch.bfloat16)
    s = torch.exp2(torch.randint(-60, 30, (m, 1), generator=torch.Generator().manual_seed(1)).double()).to(dev)
    c.x = (c.x.double() * s).to(torch.bfloat16)
    _, g, u = gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, save=True, out_dtype=torch.float32)
    _, rg, ru = c.front(0)
    assert worst_row(g, rg) <= PRODUCT and worst_row(u, ru) <= PRODUCT
    c.dh = (c.dh.double() * s).to(torch.bfloat16)
    dx = gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k, dx_dtype=torch.float32)["dx"]
    assert worst_row(dx, c.grads(0)[0]) <= PRODUCT


@pytest.mark.parametrize("m", [3, 40, 200])
@pytest.mark.parametrize("size", [-112, -60, 60, 117])
def test_sizes_of_gradients(dev, m, size):
    """dh of any size that leaves dx a normal fp32: its row's power of two takes it into fp16 and back.  2^size times 0.1 e^N(0,1),
    u act'(g) of 1.5: dg 2^-115 (normal: 2^-126) to 2^120; dx of one to a few times that."""
    import gq
    fmt, n, k = O.Q8_0, 200, 256
    c = Case(dev, fmt, m, n, k, seed=11, dtype=torch.float32)
    c.dh *= 2.0 ** size
    out = gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k, want_dgu=False)
    assert worst_row(out["dx"], c.grads(0)[0]) <= PRODUCT + half_step(torch.float32)


@pytest.mark.parametrize("m", [2, 16, 40, 200])
@pytest.mark.parametrize("bad", [np.nan, np.inf, -np.inf])
def test_nonfinite_rows(dev, m, bad):
    """A row with an Inf or NaN comes out non-finite, the others as without it."""
    import gq
    fmt, n, k = O.Q4_K, 64, 512
    c = Case(dev, fmt, m, n, k, seed=13, dtype=torch.float32)
    ref = gq.ffn_gate_up(fmt, *c.packed, c.x, n, k)
    gref = gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k)["dx"]
    c.x[1, 100] = bad
    c.dh[1, 33] = bad
    h = gq.ffn_gate_up(fmt, *c.packed, c.x, n, k)
    dx = gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k)["dx"]
    keep = [i for i in range(m) if i != 1]
    for a, b in ((h, ref), (dx, gref)):
        assert not bool(a[1].isfinite().any())
        assert torch.equal(a[keep], b[keep])


def test_extreme_gates(dev):
    """Gates where the sigmoid is 0 or 1 and where powers of g overflow: finite outputs, right limits."""
    import gq
    fmt, k = O.Q4_0, 64
    g = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 20., -20., 89., -89., 1e4, -1e4, 1e20, -1e20, 3e38, -3e38], device=dev)[None]
    n = g.shape[1]
    c = Case(dev, fmt, 1, n, k, dtype=torch.float32)
    one = torch.ones_like(g)
    for act in (0, 1):
        out = gq.ffn_gate_up_bwd(fmt, *c.packed, one, g, one, n, k, act=act)
        f, d = act_grad(act, g.double().clamp(-1e5, 1e5))
        f = torch.where(g.abs() > 1e5, g.double() * (g > 0), f)
        assert bool(((out["dg"].double() - d).abs() <= 1e-5).all())
        assert bool(((out["du"].double() - f).abs() <= 1e-5 * g.double().abs()).all())


@pytest.mark.parametrize("act", [0, 1])
def test_gradient_against_differences(dev, act):
    """dx against differences of the operator's own forward pass along a direction."""
    import gq
    fmt, m, n, k = O.Q8_0, 24, 96, 256
    c = Case(dev, fmt, m, n, k, seed=17, dtype=torch.float32)
    v = torch.randn(m, k, generator=torch.Generator().manual_seed(2)).to(dev) * c.x.abs().mean()

    def loss(x):
        return float((gq.ffn_gate_up(fmt, *c.packed, x, n, k, act=act).double() * c.dh.double()).sum())

    _, g, u = gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, act=act, save=True)
    dx = gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, g, u, n, k, act=act)["dx"]
    e = 2.0 ** -5
    along = float((dx.double() * v.double()).sum())
    # (curvature: e^2 / 6 of a third derivative of the size of the first; fp16 roundings of 3e-4 over a step of 1/32
    # of x: 1e-2; both against the norms, not the cancelled sum)
    scale = float(dx.double().norm() * v.double().norm())
    assert abs((loss(c.x + e * v) - loss(c.x - e * v)) / (2 * e) - along) <= 2e-2 * scale


def test_streams_and_workspaces(dev):
    """Calls that overlap on two streams, with workspaces of their own and without."""
    import gq
    fmt, n, k = O.Q4_K, 1024, 1024
    cases = [Case(dev, fmt, m, n, k, seed=m) for m in (3, 16, 60, 300)]
    ref = [(gq.ffn_gate_up(fmt, *c.packed, c.x, n, k), gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k)) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    ws = [gq.Workspace(dev) for _ in range(2)]
    outs = []
    for i in range(12):
        s, c = i % 2, cases[i % 4]
        with torch.cuda.stream(streams[s]):
            w = ws[s] if i < 6 else None
            outs.append((i % 4, gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, workspace=w),
                         gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k, workspace=w)))
    torch.cuda.synchronize()
    for i, h, b in outs:
        assert torch.equal(h, ref[i][0])
        for name in ("dx", "dg", "du"):
            assert torch.equal(b[name], ref[i][1][name]), name


@pytest.mark.parametrize("m", [1, 16, 64, 300])
def test_captured(dev, m):
    """A forward and backward pass in a graph, replayed on new inputs with eager work between the replays."""
    import gq
    fmt, n, k = O.Q6_K, 520, 1024
    c = Case(dev, fmt, m, n, k, seed=m)
    ws = gq.Workspace(dev, max(gq.ffn_gate_up_workspace_bytes(fmt, m, n, k), gq.ffn_gate_up_bwd_workspace_bytes(fmt, m, n, k)))
    h, g, u = (torch.empty(m, n, dtype=torch.bfloat16, device=dev) for _ in range(3))
    dg, du, dx = torch.empty_like(h), torch.empty_like(h), torch.empty(m, k, dtype=torch.bfloat16, device=dev)

    def step():
        gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, h=h, g=g, u=u, workspace=ws)
        gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, g, u, n, k, dg=dg, du=du, dx=dx, workspace=ws)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        c.x.copy_(Case(dev, fmt, m, n, k, seed=100 + i).x)
        for t in (h, g, u, dg, du, dx):
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (h, g, u, dg, du, dx)]
        step()
        torch.cuda.synchronize()
        for a, b in zip(got, (h, g, u, dg, du, dx)):
            assert torch.equal(a, b)
        c.g, c.u = g.clone(), u.clone()
        check_front(c, 0, (h, g, u), torch.bfloat16)
        check_grads(c, 0, {"dg": dg, "du": du, "dx": dx}, torch.bfloat16)


def test_repeatable(dev):
    import gq
    fmt, n, k = O.Q4_0, 3000, 2048
    for m in (1, 30, 333):
        c = Case(dev, fmt, m, n, k, seed=m)
        first = gq.ffn_gate_up(fmt, *c.packed, c.x, n, k), gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k)["dx"]
        for _ in range(3):
            assert torch.equal(gq.ffn_gate_up(fmt, *c.packed, c.x, n, k), first[0])
            assert torch.equal(gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k)["dx"], first[1])


def test_small_workspace_is_refused(dev):
    import gq
    fmt, m, n, k = O.Q4_0, 300, 512, 512
    c = Case(dev, fmt, m, n, k)
    lib = gq.load()
    for size, call in (
            (gq.ffn_gate_up_workspace_bytes(fmt, m, n, k), lambda w, b: lib.gq_ffn_gate_up(
                fmt, c.packed[0].data_ptr(), c.packed[1].data_ptr(), c.x.data_ptr(), gq.DT_BF16, c.g.data_ptr(), gq.DT_BF16,
                None, None, m, n, k, 0, w, b, None)),
            (gq.ffn_gate_up_bwd_workspace_bytes(fmt, m, n, k), lambda w, b: lib.gq_ffn_gate_up_bwd(
                fmt, c.packed[0].data_ptr(), c.packed[1].data_ptr(), c.dh.data_ptr(), c.g.data_ptr(), c.u.data_ptr(),
                gq.DT_BF16, None, None, c.x.data_ptr(), gq.DT_BF16, m, n, k, 0, w, b, None))):
        assert size > 0
        ws = torch.empty(size, dtype=torch.uint8, device=dev)
        torch.cuda.synchronize()
        assert call(ws.data_ptr(), size - 1) == 4
        assert call(ws.data_ptr(), size) == 0
        torch.cuda.synchronize()


def test_blocks_of_fewer_rows(dev):
    """Rows so long that a block holds fewer than 256 of them: three blocks, the last one ragged, scratch of the call's own."""
    import gq
    m, n, k = 300, 20, 1 << 18
    c = Case(dev, O.Q4_K, m, n, k, seed=1)
    check_front(c, 0, gq.ffn_gate_up(O.Q4_K, *c.packed, c.x, n, k, save=True), torch.bfloat16)
    m, n, k = 500, 1 << 17, 32
    c = Case(dev, O.Q4_0, m, n, k, seed=2)
    check_grads(c, 0, gq.ffn_gate_up_bwd(O.Q4_0, *c.packed, c.dh, c.g, c.u, n, k), torch.bfloat16)


@pytest.mark.parametrize("dtype", DTYPES)
def test_no_columns_between(dev, dtype):
    """N = 0: dx is a sum of nothing."""
    import gq
    m, k = 5, 256
    e, w = torch.empty(m, 0, dtype=dtype, device=dev), torch.empty(0, dtype=torch.uint8, device=dev)
    dx = torch.full((m + 1, k), 7.0, dtype=dtype, device=dev)
    out = gq.ffn_gate_up_bwd(O.Q8_0, w, w, e, e, e, 0, k, dx=dx[:m])
    assert bool((dx[:m] == 0).all()) and bool((dx[m:] == 7).all()) and out["dg"].shape == (m, 0)
    assert gq.ffn_gate_up(O.Q8_0, w, w, dx[:m], 0, k).shape == (m, 0)
    x = torch.empty(0, k, dtype=dtype, device=dev)
    full = Case(dev, O.Q8_0, 1, 16, k).packed
    assert gq.ffn_gate_up(O.Q8_0, *full, x, 16, k).shape == (0, 16)


def test_capture_without_a_workspace(dev):
    """A call that needs a workspace takes none of its own while its stream is captured; one that needs none is captured."""
    import gq
    fmt, n, k = O.Q4_K, 64, 512
    c, few = Case(dev, fmt, 40, n, k), Case(dev, fmt, 3, n, k)
    h = torch.empty(3, n, dtype=torch.bfloat16, device=dev)
    ref = gq.ffn_gate_up(fmt, *few.packed, few.x, n, k)
    out, dx = torch.empty(40, n, dtype=torch.bfloat16, device=dev), torch.empty_like(c.x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(gq.GQError):
            gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, h=out)
        with pytest.raises(gq.GQError):
            gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k, dx=dx, want_dgu=False)
        gq.ffn_gate_up(fmt, *few.packed, few.x, n, k, h=h)
    for _ in range(3):
        h.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(h, ref)


def test_block_trains_and_decodes(dev):
    """The operators as they are used together: a prompt through the block's front and the down projection, the
    backward pass of both ends, then single tokens that agree with the prompt's rows and with the f32 decode front."""
    import gq
    fmt, m, n, k = O.Q8_0, 70, 768, 512
    c = Case(dev, fmt, m, n, k, seed=23)
    down = O.gen_weights(fmt, k, n, seed=99)
    pd = gq.repack(fmt, torch.from_numpy(down).to(dev), k, n)
    wd = torch.from_numpy(O.dequant(fmt, down).reshape(k, n)).to(dev).double()
    h, g, u = gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, save=True)
    y = gq.gemm(fmt, pd, h, k, n, out_dtype=torch.bfloat16)
    assert worst_row(y, h.double() @ wd.t().contiguous()) <= PRODUCT + half_step(torch.bfloat16)
    c.g, c.u, c.dh = g, u, (torch.randn(m, k, device=dev) @ wd.float() * 0.01).to(torch.bfloat16)
    check_grads(c, 0, gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, g, u, n, k), torch.bfloat16)
    for i in (0, 33, 69):
        one = gq.ffn_gate_up(fmt, *c.packed, c.x[i], n, k, out_dtype=torch.float32)
        dec = gq.gemv_swiglu(fmt, *c.packed, c.x[i].float(), n, k)
        c1 = Case.__new__(Case)
        c1.w, c1.x = c.w, c.x[i:i + 1]
        for t in (one, dec, h[i:i + 1]):
            check_front(c1, 0, (t, None, None), t.dtype)


def test_sizes_kept_are_bounded(dev):
    """Calls of ever new lengths leave no record of each behind."""
    import gq

    def held():
        return sum(len(v) for v in vars(gq).values() if isinstance(v, (dict, list, set))) + sum(
            v.cache_info().currsize for v in vars(gq).values() if hasattr(v, "cache_info"))

    fmt, n, k = O.Q4_0, 16, 64
    c = Case(dev, fmt, 2500, n, k)
    ws, before = gq.Workspace(dev), held()
    for m in range(1, 2501):
        gq.ffn_gate_up(fmt, *c.packed, c.x[:m], n, k, workspace=ws)
    assert held() - before <= 1024


def test_a_given_stream_owns_the_outputs(dev):
    """Outputs made for a call on another stream do not lie in memory that queued work of the current one still writes."""
    import gq
    fmt, m, n, k = O.Q8_0, 64, 2048, 512
    c = Case(dev, fmt, m, n, k, seed=31)
    ref = gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, save=True)
    gref = gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k)
    q, s = torch.full((n, k // 2), 0x5A, dtype=torch.uint8, device=dev), torch.ones(n, k // 128, dtype=torch.float16, device=dev)
    wref = gq.w4_pack(q, s, None, n, k, 128)
    yref, href = gq.w4_gemv(wref, 128, c.x[:16], n, k), gq.w4_gate_up(wref, wref, 128, c.x[:16], n, k)
    side, a = torch.cuda.Stream(), torch.randn(8192, 8192, device=dev).to(torch.bfloat16)
    calls = [(lambda: gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, save=True, stream=side), ref),
             (lambda: tuple(gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k, stream=side).values()), tuple(gref.values())),
             (lambda: (gq.w4_pack(q, s, None, n, k, 128, stream=side),), (wref,)),
             (lambda: (gq.w4_gemv(wref, 128, c.x[:16], n, k, stream=side),), (yref,)),
             (lambda: (gq.w4_gate_up(wref, wref, 128, c.x[:16], n, k, stream=side),), (href,))]
    for call, want in calls:
        b = torch.mm(a, a)
        torch.cuda.synchronize()
        old = [torch.empty_like(t) for t in want for _ in range(2)]
        for _ in range(20):
            torch.mm(a, a, out=b)  # (some milliseconds of work in front of the writes)
        for t in old:
            t.fill_(77)
        del old, t
        got = call()
        side.synchronize()
        torch.cuda.synchronize()
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_a_stream_of_another_device_is_refused(dev):
    import types

    import gq
    c = Case(dev, O.Q8_0, 4, 64, 256)
    with pytest.raises(gq.GQError, match="cuda:7"):
        gq.ffn_gate_up(O.Q8_0, *c.packed, c.x, 64, 256, stream=types.SimpleNamespace(device=torch.device("cuda:7"), cuda_stream=0))


def test_a_workspace_elsewhere_is_refused(dev):
    """No kernel gets the address of host memory, or of another device's."""
    import gq
    fmt, n, k = O.Q8_0, 64, 256
    for m in (4, 40):
        c = Case(dev, fmt, m, n, k)
        with pytest.raises(gq.GQError, match="workspace"):
            gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, workspace=gq.Workspace("cpu"))
        with pytest.raises(gq.GQError, match="workspace"):
            gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k, workspace=gq.Workspace("cpu"))


def test_a_workspace_outgrown_after_a_capture(dev):
    """A captured call's workspace is not given to others when a later call needs a larger one."""
    import gq
    fmt, m, n, k = O.Q4_K, 64, 512, 4096
    c, big = Case(dev, fmt, m, n, k, seed=1), Case(dev, fmt, 900, n, k, seed=2)
    need = max(gq.ffn_gate_up_workspace_bytes(fmt, m, n, k), gq.ffn_gate_up_bwd_workspace_bytes(fmt, m, n, k))
    ws = gq.Workspace(dev, need)
    h, dx = torch.empty(m, n, dtype=torch.bfloat16, device=dev), torch.empty(m, k, dtype=torch.bfloat16, device=dev)

    def step():
        gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, h=h, workspace=ws)
        gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k, dx=dx, want_dgu=False, workspace=ws)

    step()
    torch.cuda.synchronize()
    ref = h.clone(), dx.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    size = ws.buf.numel()
    gq.ffn_gate_up(fmt, *big.packed, big.x, n, k, workspace=ws)
    gq.ffn_gate_up_bwd(fmt, *big.packed, big.dh, big.g, big.u, n, k, workspace=ws)
    assert ws.buf.numel() > size
    torch.cuda.synchronize()
    others = [torch.full((size,), 7, dtype=torch.uint8, device=dev) for _ in range(3)]
    for _ in range(3):
        h.fill_(float("nan"))
        dx.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(h, ref[0]) and torch.equal(dx, ref[1])
        assert all(bool((t == 7).all()) for t in others)
