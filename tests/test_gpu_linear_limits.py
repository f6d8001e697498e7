"""The product with its epilogue and its backward pass where they could go wrong: every tile the rule takes, long rows, types, outputs
wanted alone, ends of buffers, sizes of values, rows with an Inf or NaN, streams, graphs, workspaces, threads.

Tolerances are those of test_gpu_linear."""
import pytest
import torch

import oracle as O
from linear_ref import act_grad
from test_gpu_linear import DTYPES, FMTS, Case, check_forward, check_grads

pytestmark = pytest.mark.gpu


def rows_of(c, rows):
    """The case as if it had these rows alone."""
    r = Case.__new__(Case)
    r.fmt, r.n, r.k, r.packed, r.w, r.bias = c.fmt, c.n, c.k, c.packed, c.w, c.bias
    r.x, r.z, r.dy, r.resid = c.x[rows], c.z[rows], c.dy[rows], None if c.resid is None else c.resid[rows]
    r.m = len(r.x)
    return r


def forward(c, act=0, **kw):
    import gq
    return gq.linear(c.fmt, c.packed, c.x, c.n, c.k, bias=c.bias, act=act, resid=c.resid, **kw)


def backward(c, act=0, **kw):
    import gq
    return gq.linear_bwd(c.fmt, c.packed, c.dy, c.z, c.n, c.k, act=act, want_dbias=True, **kw)


# formats with blocks of 32: K that is no whole chunk of the layout, and an odd number of them
@pytest.mark.parametrize("fmt", [O.Q4_0, O.Q8_0])
@pytest.mark.parametrize("m,n,k", [(1, 16, 32), (3, 33, 608), (4, 40, 96), (14, 70, 416), (20, 65, 160), (50, 65, 4128), (100, 70, 4128),
                                   (300, 129, 224), (20, 100, 288), (20, 100, 8288), (130, 300, 2144), (130, 9000, 160)])
def test_short_chunks(dev, fmt, m, n, k):
    for dtype in (torch.float16, torch.bfloat16):
        c = Case(dev, fmt, m, n, k, seed=k, dtype=dtype)
        check_forward(c, 3, *forward(c, 3, save=True), dtype)
        check_grads(c, 2, backward(c, 2), dtype)


# few rows of wide and of long matrices, each tile of the rule with K in parts and without, many rows
@pytest.mark.parametrize("fmt", [O.Q4_0, O.Q8_0, O.Q4_K, O.Q6_K])
@pytest.mark.parametrize("m,n,k", [(1, 4099, 4096), (1, 9003, 1024), (2, 1500, 14336), (3, 5001, 2048), (11, 5003, 4096), (4, 300, 16128), (4, 100, 20480), (7, 1030, 8192), (12, 2100, 1024), (16, 14336, 256),
                                   (16, 100, 20480), (24, 600, 14336), (40, 3001, 2048), (40, 17000, 256), (64, 260, 4352), (90, 1500, 2304),
                                   (200, 4100, 1024), (200, 14000, 512), (260, 9000, 8192), (700, 13000, 512), (2050, 520, 512), (1500, 2100, 4096),
                                   (6000, 4100, 512), (200, 20000, 1024), (300, 520, 8192), (65, 20000, 4096), (512, 4100, 14336),
                                   (130, 14000, 8192)])
def test_large(dev, fmt, m, n, k):
    c = Case(dev, fmt, m, n, k, seed=n, dtype=torch.bfloat16)
    check_forward(c, 1, *forward(c, 1, save=True), torch.bfloat16)
    check_grads(c, 1, backward(c, 1), torch.bfloat16)


@pytest.mark.parametrize("fmt", [O.Q8_0, O.Q6_K])
@pytest.mark.parametrize("m,n,k", [(5, 100, 512), (16, 1000, 4096), (60, 500, 2048), (400, 300, 1024), (5000, 64, 8192)])
def test_fp16_rows_as_they_are(dev, fmt, m, n, k):
    """fp16 rows of whole chunks enter the products unconverted: the same from 2-byte aligned memory, where they are copied."""
    c = Case(dev, fmt, m, n, k, seed=2, dtype=torch.float16)
    y, z = forward(c, 2, save=True)
    check_forward(c, 2, y, z, torch.float16)
    odd = torch.empty(m * k + 1, dtype=torch.float16, device=dev)[1:].view(m, k).copy_(c.x)
    ref, c.x = c.x, odd
    got = forward(c, 2, save=True)
    check_forward(c, 2, *got, torch.float16)
    c.x = ref


@pytest.mark.parametrize("xdt", DTYPES)
@pytest.mark.parametrize("ydt", DTYPES)
@pytest.mark.parametrize("m", [1, 8, 40, 150])
def test_types(dev, xdt, ydt, m):
    fmt, n, k = O.Q4_K, 272, 512
    c = Case(dev, fmt, m, n, k, seed=m % 3, dtype=xdt)  # (the bias's type goes with the seed)
    c.resid = c.resid.to(ydt)
    y, z = forward(c, 2, out_dtype=ydt, save=True)
    assert y.dtype == z.dtype == ydt
    check_forward(c, 2, y, z, ydt)
    out = backward(c, 0, dx_dtype=ydt)
    assert out["dx"].dtype == ydt and out["dz"].dtype == xdt and out["dbias"].dtype == torch.float32
    check_grads(c, 0, out, xdt)


@pytest.mark.parametrize("m", [1, 4, 16, 33, 260])
def test_wanted_outputs_alone(dev, m):
    """Each output by itself gives what it gives with the others; y over the residual, dz over dy or z."""
    import gq
    fmt, n, k = O.Q8_0, 100, 256
    c = Case(dev, fmt, m, n, k, seed=5)
    for act in (0, 1, 2, 3):
        y, z = forward(c, act, save=True)
        assert torch.equal(forward(c, act), y)
        kept = c.resid.clone()
        into = gq.linear(fmt, c.packed, c.x, n, k, bias=c.bias, act=act, resid=kept, y=kept)
        assert into is kept and torch.equal(kept, y)
        full = backward(c, act)
        for alone in ("dx", "dz", "dbias"):
            part = gq.linear_bwd(fmt, c.packed, c.dy, c.z, n, k, act=act, want_dx=alone == "dx", want_dz=alone == "dz",
                                 want_dbias=alone == "dbias")
            for name in full:
                assert part[name] is None if name != alone else torch.equal(part[name], full[name])
        for over in ("dy", "z"):
            dy, zz = c.dy.clone(), c.z.clone()
            out = gq.linear_bwd(fmt, c.packed, dy, zz, n, k, act=act, dz=dy if over == "dy" else zz, want_dbias=True)
            assert all(torch.equal(out[name], full[name]) for name in full)
    none = gq.linear_bwd(fmt, c.packed, c.dy, None, n, k, want_dbias=True)
    assert torch.equal(none["dz"], c.dy)
    check_grads(c, gq.ACT_NONE, none, torch.bfloat16)
    plain = gq.linear(fmt, c.packed, c.x, n, k)  # no bias, no residual: the product alone
    c.bias = c.resid = None
    check_forward(c, gq.ACT_NONE, plain, plain, torch.bfloat16)


def test_one_row_without_its_dimension(dev):
    import gq
    c = Case(dev, O.Q4_0, 1, 96, 256, seed=4)
    y = gq.linear(O.Q4_0, c.packed, c.x[0], 96, 256, bias=c.bias)
    assert y.shape == (1, 96) and torch.equal(y, gq.linear(O.Q4_0, c.packed, c.x, 96, 256, bias=c.bias))


@pytest.mark.parametrize("m", [1, 4, 5, 16, 20, 64, 100, 300])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("fmt,k", [(O.Q4_0, 288), (O.Q8_0, 256)])
def test_nothing_behind_the_outputs(dev, m, dtype, fmt, k):
    """Values before and behind the outputs stay as they were, at any alignment of the operands."""
    import gq
    n = 101
    c = Case(dev, fmt, m, n, k, seed=9, dtype=dtype)

    def guarded(rows, cols, at, dt=dtype):
        buf = torch.full((at + rows * cols + 2000,), 7.0, dtype=dt, device=dev)
        return buf, buf[at:at + rows * cols].view(rows, cols)

    for at in (0, 1, 3):
        bufs, outs = zip(*[guarded(m, cols, at) for cols in (n, n, n, k)], guarded(1, n, at, torch.float32))
        x = guarded(m, k, at)[1].copy_(c.x)
        resid, dy, z = (guarded(m, n, at)[1].copy_(t) for t in (c.resid, c.dy, c.z))
        bias = guarded(1, n, at, c.bias.dtype)[1][0].copy_(c.bias)
        gq.linear(fmt, c.packed, x, n, k, bias=bias, act=0, resid=resid, y=outs[0], z=outs[1])
        check_forward(c, 0, *outs[:2], dtype)
        gq.linear_bwd(fmt, c.packed, dy, z, n, k, act=1, dz=outs[2], dx=outs[3], dbias=outs[4][0])
        check_grads(c, 1, {"dz": outs[2], "dx": outs[3], "dbias": outs[4][0]}, dtype)
        for buf, o in zip(bufs, outs):
            assert bool((buf[:at] == 7).all()) and bool((buf[at + o.numel():] == 7).all())


@pytest.mark.parametrize("m", [1, 8, 48, 200])
def test_sizes_of_rows(dev, m):
    """Rows far outside fp16's range, in both directions, keep their precision."""
    fmt, n, k = O.Q8_0, 128, 512
    c = Case(dev, fmt, m, n, k, seed=11, dtype=torch.bfloat16, bias=False, resid=False)
    s = torch.exp2(torch.randint(-60, 30, (m, 1), generator=torch.Generator().manual_seed(1)).double()).to(dev)
    c.x = (c.x.double() * s).to(torch.bfloat16)
    y = forward(c, 2, out_dtype=torch.float32)
    check_forward(c, 2, y, y, torch.float32)
    c.dy = (c.dy.double() * s).to(torch.bfloat16)
    check_grads(c, 0, backward(c, 0, dx_dtype=torch.float32, want_dz=False), torch.bfloat16)


@pytest.mark.parametrize("fmt", [O.Q4_0, O.Q8_0, O.Q4_K, O.Q6_K])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k", [(1, 512), (4, 1280), (11, 2304), (24, 2304), (80, 512)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_nonfinite_rows(dev, fmt, dtype, m, k, bad):
    """A row with an Inf or NaN comes out non-finite, the others as without it."""
    n = 200
    c = Case(dev, fmt, m, n, k, seed=13, dtype=dtype)
    keep = [i for i in range(m) if i != m // 2]
    ref, gref = forward(c, 2, save=True), backward(c, 2)
    c.x[m // 2, 100] = bad
    c.dy[m // 2, 33] = bad
    got, gout = forward(c, 2, save=True), backward(c, 2)
    for a, b in zip((*got, gout["dx"], gout["dz"]), (*ref, gref["dx"], gref["dz"])):
        assert torch.equal(a[keep], b[keep])
    for a in (*got, gout["dx"]):
        assert not bool(a[m // 2].isfinite().any())
    assert not bool(gout["dz"][m // 2, 33].isfinite()) and not bool(gout["dbias"][33].isfinite())
    at = [i for i in range(n) if i != 33]
    assert bool(gout["dbias"][at].isfinite().all())


@pytest.mark.parametrize("m", [1, 8, 40])
def test_extreme_sums(dev, m):
    """Sums (of zero weights: the bias) where the sigmoid is 0 or 1 and where powers overflow: right limits, and a NaN stays one."""
    import gq
    fmt, k = O.Q4_0, 64
    g = torch.tensor([0.0, -0.0, 1e-30, -1e-30, 20., -20., 89., -89., 1e4, -1e4, 1e20, -1e20, 3e38, -3e38, float("nan")], device=dev)
    n = g.shape[0]
    packed = gq.repack(fmt, torch.zeros(n * k // 32 * 18, dtype=torch.uint8, device=dev), n, k)
    x, one = torch.ones(m, k, device=dev), torch.ones(m, n, device=dev)
    for act in (0, 1, 2, 3):
        y = gq.linear(fmt, packed, x, n, k, bias=g, act=act)
        dz = gq.linear_bwd(fmt, packed, one, g.repeat(m, 1), n, k, act=act)["dz"]
        f, d = act_grad(act, g.double().clamp(-1e5, 1e5))
        if act != gq.ACT_NONE:
            f = torch.where(g.abs() > 1e5, g.double() * (g > 0), f)
        else:
            f = g.double()
        assert bool(y[:, -1].isnan().all())
        assert bool(((y[:, :-1].double() - f[:-1]).abs() <= 1e-5 * g[:-1].double().abs()).all())
        assert bool(((dz[:, :-1].double() - d[:-1]).abs() <= 1e-5).all())


@pytest.mark.parametrize("act", [0, 1, 2])
def test_gradient_against_differences(dev, act):
    """dx and dbias against differences of the operator's own forward pass along a direction."""
    import gq
    fmt, m, n, k = O.Q8_0, 24, 96, 256
    c = Case(dev, fmt, m, n, k, seed=18, dtype=torch.float32)
    gen = torch.Generator().manual_seed(2)
    v = torch.randn(m, k, generator=gen).to(dev) * c.x.abs().mean()
    b = torch.randn(n, generator=gen).to(dev)

    def loss(x, bias):
        return float((gq.linear(fmt, c.packed, x, n, k, bias=bias, act=act, resid=c.resid).double() * c.dy.double()).sum())

    bias = c.bias.float()
    c.z = gq.linear(fmt, c.packed, c.x, n, k, bias=bias, act=act, save=True)[1]
    out = backward(c, act)
    e = 2.0 ** -5
    # (curvature: e^2 / 6 of a third derivative of the size of the first; fp16 roundings of 3e-4 over a step of 1/32: 1e-2;
    # both against the norms, not the cancelled sum)
    along, scale = float((out["dx"].double() * v.double()).sum()), float(out["dx"].double().norm() * v.double().norm())
    assert abs((loss(c.x + e * v, bias) - loss(c.x - e * v, bias)) / (2 * e) - along) <= 2e-2 * scale
    along, scale = float((out["dbias"].double() * b.double()).sum()), float(out["dz"].double().norm() * b.double().norm() * m ** 0.5)
    assert abs((loss(c.x, bias + e * b) - loss(c.x, bias - e * b)) / (2 * e) - along) <= 2e-2 * scale


def test_streams_and_workspaces(dev):
    """Calls that overlap on two streams, with workspaces of their own and without."""
    import gq
    fmt, n, k = O.Q4_K, 1024, 4096
    cases = [Case(dev, fmt, m, n, k, seed=m) for m in (3, 16, 60, 300)]
    ref = [(forward(c), backward(c)) for c in cases]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    ws = [gq.Workspace(dev) for _ in range(2)]
    outs = []
    for i in range(12):
        s, c = i % 2, cases[i % 4]
        with torch.cuda.stream(streams[s]):
            w = ws[s] if i < 6 else None
            outs.append((i % 4, forward(c, workspace=w), backward(c, workspace=w)))
    torch.cuda.synchronize()
    for i, y, b in outs:
        assert torch.equal(y, ref[i][0])
        for name in ("dx", "dz", "dbias"):
            assert torch.equal(b[name], ref[i][1][name]), name


@pytest.mark.parametrize("m", [1, 16, 64, 300])
def test_captured(dev, m):
    """A forward and backward pass in a graph, replayed on new inputs with eager work between the replays."""
    import gq
    fmt, n, k = O.Q6_K, 520, 4096
    c = Case(dev, fmt, m, n, k, seed=m)
    ws = gq.Workspace(dev, max(gq.linear_workspace_bytes(fmt, m, n, k), gq.linear_bwd_workspace_bytes(fmt, m, n, k)))
    y, z, dz = (torch.empty(m, n, dtype=torch.bfloat16, device=dev) for _ in range(3))
    dx, db = torch.empty(m, k, dtype=torch.bfloat16, device=dev), torch.empty(n, device=dev)

    def step():
        gq.linear(fmt, c.packed, c.x, n, k, bias=c.bias, act=0, resid=c.resid, y=y, z=z, workspace=ws)
        gq.linear_bwd(fmt, c.packed, c.dy, z, n, k, act=0, dz=dz, dx=dx, dbias=db, workspace=ws)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        c.x.copy_(Case(dev, fmt, m, n, k, seed=100 + i).x)
        for t in (y, z, dz, dx, db):
            t.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (y, z, dz, dx, db)]
        step()
        torch.cuda.synchronize()
        for a, b in zip(got, (y, z, dz, dx, db)):
            assert torch.equal(a, b)
        c.z = z.clone()
        check_forward(c, 0, y, z, torch.bfloat16)
        check_grads(c, 0, {"dz": dz, "dx": dx, "dbias": db}, torch.bfloat16)


def test_repeatable(dev):
    fmt, n, k = O.Q4_0, 3000, 4096
    for m in (1, 12, 30, 333):
        c = Case(dev, fmt, m, n, k, seed=m)
        first, grads = forward(c), backward(c)
        for _ in range(3):
            assert torch.equal(forward(c), first)
            again = backward(c)
            assert all(torch.equal(again[name], grads[name]) for name in grads)


@pytest.mark.parametrize("most,n,k", [(65, 2048, 512), (300, 1000, 1024), (96, 520, 4352), (20, 300, 20480)])
def test_a_workspace_for_more_rows_serves_fewer(dev, most, n, k):
    """The bytes given for `most` rows are taken for every call of fewer, one byte less is refused, and nothing is written behind them."""
    import gq
    fmt, lib = O.Q4_0, gq.load()
    c = Case(dev, fmt, most, n, k, seed=7, bias=False, resid=False)
    s = torch.cuda.current_stream().cuda_stream
    for back, size in ((False, gq.linear_workspace_bytes), (True, gq.linear_bwd_workspace_bytes)):
        need = size(fmt, most, n, k)
        buf = torch.full((need + 65536,), 7, dtype=torch.uint8, device=dev)
        for m in sorted({1, 4, 5, 17, 31, 32, 33, 63, 64, most - 1, most} & set(range(1, most + 1))):
            f, db = rows_of(c, slice(0, m)), torch.empty(n, device=dev)
            out = torch.empty(m, k if back else n, dtype=torch.bfloat16, device=dev)

            def call(nbytes):
                if back:
                    return lib.gq_linear_bwd(fmt, c.packed.data_ptr(), c.dy.data_ptr(), c.z.data_ptr(), gq.DT_BF16, 0, None,
                                             out.data_ptr(), gq.DT_BF16, db.data_ptr(), m, n, k, buf.data_ptr(), nbytes, s)
                return lib.gq_linear(fmt, c.packed.data_ptr(), c.x.data_ptr(), gq.DT_BF16, None, 0, 2, None, out.data_ptr(),
                                     gq.DT_BF16, None, m, n, k, buf.data_ptr(), nbytes, s)

            if back or m > 4:
                assert call(size(fmt, m, n, k) - 1) == 4
            assert call(need) == 0
            if back:
                check_grads(f, 0, {"dx": out, "dz": None, "dbias": db}, torch.bfloat16)
            else:
                check_forward(f, 2, out, out, torch.bfloat16)
            assert bool((buf[need:] == 7).all())


def test_blocks_of_fewer_rows(dev):
    """Rows so long that a block holds fewer than 256 of them: the last one ragged, scratch of the call's own."""
    m, n, k = 300, 20, 1 << 18
    c = Case(dev, O.Q4_K, m, n, k, seed=1)
    check_forward(c, 0, *forward(c, 0, save=True), torch.bfloat16)
    c = Case(dev, O.Q8_0, m, n, k, seed=2, dtype=torch.float16)
    check_forward(c, 0, *forward(c, 0, save=True), torch.float16)
    m, n, k = 500, 1 << 17, 32
    c = Case(dev, O.Q4_0, m, n, k, seed=3)
    check_grads(c, 0, backward(c, 0), torch.bfloat16)


def test_long_rows_of_the_bias_gradient(dev):
    """Columns so many that a workgroup keeps a part of its sums in memory, and that fewer of them share the rows."""
    m, n, k = 700, 50021, 32
    c = Case(dev, O.Q8_0, m, n, k, seed=3)
    check_grads(c, 0, backward(c, 0), torch.bfloat16)
    check_grads(c, 0, backward(c, 0, want_dx=False), torch.bfloat16)


@pytest.mark.parametrize("dtype", DTYPES)
def test_empty(dev, dtype):
    """N = 0: dx is a sum of nothing; M = 0: so is dbias."""
    import gq
    m, k = 5, 256
    e, w = torch.empty(m, 0, dtype=dtype, device=dev), torch.empty(0, dtype=torch.uint8, device=dev)
    dx = torch.full((m + 1, k), 7.0, dtype=dtype, device=dev)
    out = gq.linear_bwd(O.Q8_0, w, e, e, 0, k, dx=dx[:m], want_dbias=True)
    assert bool((dx[:m] == 0).all()) and bool((dx[m:] == 7).all()) and out["dz"].shape == (m, 0) and out["dbias"].shape == (0,)
    assert gq.linear(O.Q8_0, w, dx[:m], 0, k).shape == (m, 0)
    x = torch.empty(0, k, dtype=dtype, device=dev)
    c = Case(dev, O.Q8_0, 1, 16, k)
    assert gq.linear(O.Q8_0, c.packed, x, 16, k, bias=c.bias).shape == (0, 16)
    db = torch.full((17,), 7.0, device=dev)
    none = torch.empty(0, 16, dtype=dtype, device=dev)
    out = gq.linear_bwd(O.Q8_0, c.packed, none, none, 16, k, dbias=db[:16])
    assert out["dx"].shape == (0, k) and bool((db[:16] == 0).all()) and bool(db[16] == 7)


def test_capture_without_a_workspace(dev):
    """A call that needs a workspace takes none of its own while its stream is captured; one that needs none is captured."""
    import gq
    fmt, n, k = O.Q4_K, 64, 512
    c, few = Case(dev, fmt, 40, n, k), Case(dev, fmt, 3, n, k)
    y = torch.empty(3, n, dtype=torch.bfloat16, device=dev)
    ref = forward(few)
    out, dx = torch.empty(40, n, dtype=torch.bfloat16, device=dev), torch.empty_like(c.x)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        with pytest.raises(gq.GQError):
            forward(c, y=out)
        with pytest.raises(gq.GQError):
            gq.linear_bwd(fmt, c.packed, c.dy, c.z, n, k, dx=dx, want_dz=False)
        forward(few, y=y)
    for _ in range(3):
        y.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ref)


def test_sizes_kept_are_bounded(dev):
    """Calls of ever new lengths leave no record of each behind."""
    import gq

    def held():
        return sum(len(v) for v in vars(gq).values() if isinstance(v, (dict, list, set))) + sum(
            v.cache_info().currsize for v in vars(gq).values() if hasattr(v, "cache_info"))

    fmt, n, k = O.Q4_0, 16, 64
    c = Case(dev, fmt, 1500, n, k)
    ws, before = gq.Workspace(dev), held()
    for m in range(1, 1501):
        gq.linear(fmt, c.packed, c.x[:m], n, k, workspace=ws)
        gq.linear_bwd(fmt, c.packed, c.dy[:m], None, n, k, workspace=ws)
    assert held() - before <= 1024


def test_a_given_stream_owns_the_outputs(dev):
    """Outputs made for a call on another stream do not lie in memory that queued work of the current one still writes."""
    import gq
    fmt, m, n, k = O.Q8_0, 64, 2048, 512
    c = Case(dev, fmt, m, n, k, seed=31)
    ref, gref = forward(c, save=True), backward(c)
    side, a = torch.cuda.Stream(), torch.randn(8192, 8192, device=dev).to(torch.bfloat16)
    calls = [(lambda: forward(c, save=True, stream=side), ref),
             (lambda: tuple(backward(c, stream=side).values()), tuple(gref.values()))]
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


def test_operands_elsewhere_are_refused(dev):
    """A stream of another device, and no kernel gets the address of host memory."""
    import types

    import gq
    fmt, n, k = O.Q8_0, 64, 256
    c = Case(dev, fmt, 40, n, k)
    with pytest.raises(gq.GQError, match="cuda:7"):
        forward(c, stream=types.SimpleNamespace(device=torch.device("cuda:7"), cuda_stream=0))
    for call in (forward, backward):
        with pytest.raises(gq.GQError, match="workspace"):
            call(c, workspace=gq.Workspace("cpu"))
    for name, bad in (("bias", c.bias.cpu()), ("resid", c.resid.cpu()), ("resid", c.resid.float()), ("resid", c.resid[:39]),
                      ("bias", c.bias[:63]), ("y", c.resid.t()), ("z", c.resid.float())):
        with pytest.raises(gq.GQError, match=name):
            gq.linear(fmt, c.packed, c.x, n, k, **{name: bad})
    for name, bad in (("dx", c.x.cpu()), ("dz", c.dy.float()), ("dbias", c.bias[:5].float()), ("dbias", torch.empty(n, device=dev).half())):
        with pytest.raises(gq.GQError, match=name):
            gq.linear_bwd(fmt, c.packed, c.dy, c.z, n, k, **{name: bad})
    with pytest.raises(gq.GQError, match="w"):
        gq.linear(fmt, c.packed[:-16], c.x, n, k)
    with pytest.raises(gq.GQError, match="x"):
        gq.linear(fmt, c.packed, c.x[:, ::2], n, k // 2)
    with pytest.raises(gq.GQError):  # (a gradient through an activation needs the sums)
        gq.linear_bwd(fmt, c.packed, c.dy, None, n, k, act=gq.ACT_RELU)


def test_a_workspace_outgrown_after_a_capture(dev):
    """A captured call's workspace is not given to others when a later call needs a larger one."""
    import gq
    fmt, m, n, k = O.Q4_K, 64, 512, 4096
    c, big = Case(dev, fmt, m, n, k, seed=1), Case(dev, fmt, 900, n, k, seed=2)
    ws = gq.Workspace(dev, max(gq.linear_workspace_bytes(fmt, m, n, k), gq.linear_bwd_workspace_bytes(fmt, m, n, k)))
    y, dx = torch.empty(m, n, dtype=torch.bfloat16, device=dev), torch.empty(m, k, dtype=torch.bfloat16, device=dev)

    def step():
        forward(c, y=y, workspace=ws)
        gq.linear_bwd(fmt, c.packed, c.dy, c.z, n, k, act=0, dx=dx, want_dz=False, workspace=ws)

    step()
    torch.cuda.synchronize()
    ref = y.clone(), dx.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    size = ws.buf.numel()
    forward(big, workspace=ws)
    backward(big, workspace=ws)
    assert ws.buf.numel() > size
    torch.cuda.synchronize()
    others = [torch.full((size,), 7, dtype=torch.uint8, device=dev) for _ in range(3)]
    for _ in range(3):
        y.fill_(float("nan"))
        dx.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ref[0]) and torch.equal(dx, ref[1])
        assert all(bool((t == 7).all()) for t in others)


def test_calls_of_several_threads(dev):
    """Threads on streams of their own, without workspaces: each call's result is what it is alone."""
    import threading
    fmt, n, k = O.Q6_K, 700, 2304
    cases = [Case(dev, fmt, m, n, k, seed=m) for m in (2, 12, 70, 200)]
    want = [(forward(c), backward(c)) for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    y, g = forward(cases[i]), backward(cases[i])
                    if not torch.equal(y, want[i][0]) or not all(torch.equal(g[name], want[i][1][name]) for name in g):
                        wrong.append(i)
        except Exception as e:  # (a thread's exception would be lost)
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(cases))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_two_captured_graphs_replayed_together(dev):
    """Two graphs with workspaces of their own, replayed at once on two streams."""
    import gq
    fmt, n, k = O.Q4_K, 1024, 4352
    made = []
    for m in (40, 260):
        c, ws = Case(dev, fmt, m, n, k, seed=m), gq.Workspace(dev)
        y, dx = torch.empty(m, n, dtype=torch.bfloat16, device=dev), torch.empty(m, k, dtype=torch.bfloat16, device=dev)

        def step(c=c, ws=ws, y=y, dx=dx):
            forward(c, y=y, workspace=ws)
            gq.linear_bwd(fmt, c.packed, c.dy, c.z, n, k, act=0, dx=dx, want_dz=False, workspace=ws)

        step()
        torch.cuda.synchronize()
        want, graph = (y.clone(), dx.clone()), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        made.append((graph, torch.cuda.Stream(), (y, dx), want, step))  # (step: what the graph reads stays alive)
    for _ in range(4):
        for _, _, out, _, _ in made:
            for t in out:
                t.fill_(float("nan"))
        torch.cuda.synchronize()
        for graph, stream, _, _, _ in made:
            with torch.cuda.stream(stream):
                for _ in range(5):
                    graph.replay()
        torch.cuda.synchronize()
        for _, _, out, want, _ in made:
            assert all(torch.equal(a, b) for a, b in zip(out, want))


FAR = [0, 1, 70000, 131071, 131072, 149870, 149999]  # rows on both sides of 4 GiB of outputs, and the last


def test_past_4_gib(dev):
    """150000 x 16384 outputs of 2 bytes: 4.9 GB each."""
    fmt, m, n, k = O.Q4_0, 150000, 16384, 64
    c = Case(dev, fmt, 1000, n, k, seed=3)
    c.x = torch.randn(m, k, generator=torch.Generator().manual_seed(4)).to(dev).to(torch.bfloat16) * c.x.abs().mean()
    c.z, c.dy, c.resid = (t.repeat(150, 1) for t in (c.z, c.dy, c.resid))
    y, z = forward(c, 0, save=True)
    f = rows_of(c, FAR)
    check_forward(f, 0, y[FAR], z[FAR], torch.bfloat16)
    del y, z
    out = backward(c, 0)
    part = {"dz": out["dz"][FAR], "dx": out["dx"][FAR], "dbias": None}
    check_grads(f, 0, part, torch.bfloat16)
    d = act_grad(0, c.z[:1000].double())[1] * c.dy[:1000].double()
    assert bool(((out["dbias"].double() - 150 * d.sum(0)).abs()
                 <= 150 * 4e-6 * c.dy[:1000].double().abs().sum(0) + (m / 256 + 2) * 2 ** -24 * 150 * d.abs().sum(0)).all())


@pytest.mark.parametrize("fmt", FMTS)
def test_a_projection_adapts_and_decodes(dev, fmt):
    """The operators as they are used together: a projection with bias and activation and the one back, added to the stream in
    place, for a prompt and for single tokens, and their gradients from the last to the first."""
    import gq
    m, n, k = 37, 768, 512
    up, down = Case(dev, fmt, m, n, k, seed=23, bias=True, resid=False), Case(dev, fmt, m, k, n, seed=24, bias=False, resid=False)
    stream = (1.5 * torch.randn(m, k, generator=torch.Generator().manual_seed(1))).to(torch.bfloat16).to(dev)
    h, z = gq.linear(fmt, up.packed, up.x, n, k, bias=up.bias, act=gq.ACT_GELU_TANH, save=True)
    check_forward(up, gq.ACT_GELU_TANH, h, z, torch.bfloat16)
    y = gq.linear(fmt, down.packed, h, k, n, resid=stream, y=stream.clone())
    down.x, down.resid = h, stream
    check_forward(down, gq.ACT_NONE, y, None, torch.bfloat16)
    for i in (0, 17, 36):
        one = gq.linear(fmt, up.packed, up.x[i:i + 1], n, k, bias=up.bias, act=gq.ACT_GELU_TANH)
        check_forward(rows_of(up, slice(i, i + 1)), gq.ACT_GELU_TANH, one, None, torch.bfloat16)
        check_forward(rows_of(down, slice(i, i + 1)), gq.ACT_NONE, gq.linear(fmt, down.packed, h[i:i + 1], k, n, resid=stream[i:i + 1]), None,
                      torch.bfloat16)
    dy = (0.1 * torch.randn(m, k, generator=torch.Generator().manual_seed(2))).to(torch.bfloat16).to(dev)
    down.dy = dy
    dh = gq.linear_bwd(fmt, down.packed, dy, None, k, n)["dx"]
    check_grads(down, gq.ACT_NONE, {"dx": dh, "dz": None, "dbias": None}, torch.bfloat16)
    up.dy, up.z = dh, z
    check_grads(up, gq.ACT_GELU_TANH, gq.linear_bwd(fmt, up.packed, dh, z, n, k, act=gq.ACT_GELU_TANH, want_dbias=True), torch.bfloat16)
