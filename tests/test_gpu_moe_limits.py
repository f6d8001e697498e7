"""The mixture-of-experts layer where it could go wrong: choices between equal, masked and non-finite logits, each kernel's limits, types,
ends of buffers, sizes of values, streams, graphs, workspaces, threads, expert tensors past 4 GiB.

Tolerances are those of test_gpu_moe."""
import numpy as np
import pytest
import torch

import oracle as O
from test_gpu_moe import DTYPES, Layer, check, choose

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


def run(la, x, top, **kw):
    import gq
    return gq.moe_layer(la.fmt, *la.packed[:2], la.fmt_down, la.packed[2], la.router, x, la.n, la.k, la.e, top, **kw)


def products(la, x, ids, w, **kw):
    import gq
    return gq.moe_ffn(la.fmt, *la.packed[:2], la.fmt_down, la.packed[2], x, ids, w, la.n, la.k, la.e, **kw)


def random_choice(la, m, top, seed=0):
    gen = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(la.e, generator=gen)[:top] for _ in range(m)]).int().to(la.dev)
    return ids, torch.rand(m, top, generator=gen).to(la.dev)


def logits_as_given(l, dev):
    """x and a router whose logits are the rows of l: x of one 1, the logits in that column (0 x Inf: only finite ones, or one row)."""
    m, e = l.shape
    k = 8 * -(-max(m, 8) // 8)
    x, r = torch.zeros(m, k, device=dev), torch.zeros(e, k, device=dev)
    x[torch.arange(m), torch.arange(m)] = 1
    r[:, :m] = l.t()
    return x, r, k


@pytest.mark.parametrize("e,top", [(2, 1), (8, 3), (64, 16), (65, 4), (200, 16), (1024, 16)])
@pytest.mark.parametrize("bias", [False, True])
def test_of_equal_logits_the_lower_number(dev, e, top, bias):
    import gq
    gen = torch.Generator().manual_seed(e)
    l = torch.randint(-2, 2, (8, e), generator=gen).float().to(dev) * 0.5
    l[0] = 0
    l[1] = -0.0
    x, r, k = logits_as_given(l, dev)
    b = torch.zeros(e, device=dev) if bias else None
    ids, w = gq.moe_route(r, x, k, e, top, router_bias=b)
    rid, rw = choose(x, r, top, 0, True, 1.0, b)
    assert torch.equal(ids.long(), rid) and ids[0].tolist() == list(range(top))
    assert bool(((w.double() - rw).abs() <= 2 ** -23 * rw).all())


def test_low_words_decide(dev):
    """Logits that differ by one step of 64 bits (2^-52 of 1: products of fp32 values that cancel) are different ones."""
    import gq
    e, k = 70, 32
    x = torch.zeros(1, k, device=dev)
    x[0, 0], x[0, 1], x[0, 2] = 1, 2.0 ** -26, 2.0 ** -26
    r = torch.zeros(e, k, device=dev)
    r[:, 0] = 1
    order = torch.randperm(e, generator=torch.Generator().manual_seed(1))
    r[:, 1] = order.to(dev) * 2.0 ** -26  # (logits 1 + order 2^-52)
    ids, _ = gq.moe_route(r, x, k, e, 16)
    assert ids[0].tolist() == torch.argsort(order, descending=True)[:16].tolist()


@pytest.mark.parametrize("e", [3, 64, 130, 1000])
@pytest.mark.parametrize("score", [0, 1])
def test_masked_experts(dev, e, score):
    """Experts whose logit (with a bias: s + bias) is -Inf are never taken; all of them masked: a row of nothing."""
    import gq
    top = 3
    gen = torch.Generator().manual_seed(e)
    # one row of x of ones: every logit is a sum of the router's row
    x = torch.ones(1, 8, device=dev)
    for left in (0, 1, 2, 3, e):
        l = torch.randn(e, generator=gen)
        l[torch.randperm(e, generator=gen)[:e - left]] = -INF
        r = torch.zeros(e, 8, device=dev)
        r[:, 0] = l.to(dev)
        ids, w = gq.moe_route(r, x, 8, e, top, score=score)
        n = min(left, top)
        want = torch.sort(l, descending=True, stable=True).indices[:n]
        assert ids[0, :n].tolist() == want.tolist() and ids[0, n:].tolist() == [-1] * (top - n)
        assert bool((w[0, n:] == 0).all()) and bool((w[0, :n] > 0).all())
        s = torch.softmax(l[want].double(), 0) if score == 0 else torch.sigmoid(l[want].double())
        assert bool(((w[0, :n].double().cpu() - s / s.sum()).abs() <= 2 ** -23).all())
        # the same mask as a bias
        finite = torch.randn(e, 8, generator=gen).to(dev)
        b = torch.where(l == -INF, -INF, 0.0).float().to(dev)
        ids, w = gq.moe_route(finite, x, 8, e, top, score=score, router_bias=b)
        rid, rw = choose(x, finite, top, score, False, 1.0, b)
        assert torch.equal(ids.long()[0, :n], rid[0, :n]) and ids[0, n:].tolist() == [-1] * (top - n)
        assert bool(((w.double() - torch.nan_to_num(rw / rw.sum())).abs() <= 2 ** -23).all())


def test_masks_of_the_lowest_value(dev):
    """A mask of fp32's lowest value leaves an expert the last choice, with a weight of 0, not a NaN."""
    import gq
    e, top, low = 5, 3, torch.finfo(torch.float32).min
    x = torch.zeros(1, 8, device=dev)
    x[0, 0] = 1
    r = torch.zeros(e, 8, device=dev)
    r[:, 0] = torch.tensor([low, 0.5, low, low, low], device=dev)
    ids, w = gq.moe_route(r, x, 8, e, top)
    assert ids.tolist() == [[1, 0, 2]] and w.tolist() == [[1, 0, 0]]
    r[:, 0] = low
    ids, w = gq.moe_route(r, x, 8, e, top)
    assert ids.tolist() == [[0, 1, 2]] and bool(((w - 1 / 3).abs() <= 2 ** -24).all())
    ids, w = gq.moe_route(r, x, 8, e, top, score=gq.SCORE_SIGMOID)  # (scores of 0, and their sum: weights of 0)
    assert ids.tolist() == [[0, 1, 2]] and w.tolist() == [[0, 0, 0]]
    r[:] = 0
    b = torch.full((e,), low, device=dev)
    ids, w = gq.moe_route(r, x, 8, e, top, router_bias=b)
    assert ids.tolist() == [[0, 1, 2]] and bool(((w - 1 / 3).abs() <= 2 ** -24).all())


@pytest.mark.parametrize("bad", [NAN, INF, -INF])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m", [2, 4, 5, 33, 64])
def test_nonfinite_tokens(dev, m, dtype, bad):
    """A token with an Inf or NaN comes out non-finite, the others as without it."""
    la = Layer(dev, O.Q4_K, O.Q8_0, 6, 256, 256, seed=3)
    x = la.x(m, dtype)
    ids, w = random_choice(la, m, 2)
    ref, lref = products(la, x, ids, w), run(la, x, 2, save=True)
    x[m // 2, 100] = bad
    keep = [i for i in range(m) if i != m // 2]
    got = products(la, x, ids, w)
    assert torch.equal(got[keep], ref[keep]) and not bool(got[m // 2].isfinite().any())
    got = run(la, x, 2, save=True)
    assert all(torch.equal(a[keep], b[keep]) for a, b in zip(got, lref))
    picked = got[1][m // 2]
    assert bool(((picked >= -1) & (picked < 6)).all())
    if bool((picked >= 0).any()):
        assert not bool(got[0][m // 2].isfinite().any())


@pytest.mark.parametrize("m", [1, 2, 4, 8])
def test_nonfinite_weights(dev, m):
    """A weight of Inf or NaN reaches its own token alone."""
    la = Layer(dev, O.Q8_0, O.Q4_K, 6, 256, 256, seed=4)
    x = la.x(m, torch.bfloat16)
    ids, w = random_choice(la, m, 2)
    ref = products(la, x, ids, w)
    for bad in (NAN, INF):
        w[0, 1] = bad
        got = products(la, x, ids, w)
        assert torch.equal(got[1:], ref[1:]) and not bool(got[0].isfinite().any())


# m, e, top, n, k: rows that fill LDS and rows that do not, experts past a lane's two, rows of h of several chunks, one expert of many tokens
@pytest.mark.parametrize("fmt,down", [(O.Q4_0, O.Q8_0), (O.Q8_0, O.Q4_0), (O.Q4_K, O.Q6_K), (O.Q6_K, O.Q4_K)])
@pytest.mark.parametrize("m,e,top,n,k", [(1, 4, 2, 3584, 1024), (1, 2, 1, 256, 65536), (2, 2, 1, 256, 34048), (4, 2, 2, 256, 15872), (4, 3, 2, 256, 16128),
                                         (4, 3, 2, 256, 16384), (4, 3, 2, 8192, 256), (4, 3, 2, 8448, 256), (4, 3, 3, 8448, 256),
                                         (3, 140, 16, 256, 256), (1, 300, 16, 256, 512), (4, 17, 16, 1280, 256), (33, 1, 1, 1536, 2304), (50, 200, 16, 256, 512),
                                         (64, 64, 8, 1024, 2048), (20, 6, 2, 512, 9216)])
def test_large(dev, fmt, down, m, e, top, n, k):
    la = Layer(dev, fmt, down, e, n, k, seed=m)
    la.router *= 1 / la.size
    x = la.x(m, torch.bfloat16)
    y, ids, w = run(la, x, top, save=True)
    rid, rw = choose(x, la.router, top, 0, True, 1.0, None)
    assert torch.equal(ids.long(), rid)
    check(la, x, rid, rw, 0, None, y)


@pytest.mark.parametrize("xdt", DTYPES)
@pytest.mark.parametrize("ydt", DTYPES)
@pytest.mark.parametrize("rdt", DTYPES)
@pytest.mark.parametrize("m", [1, 3, 9])
def test_types(dev, xdt, ydt, rdt, m):
    la = Layer(dev, O.Q4_0, O.Q6_K, 9, 256, 256, seed=5, router=rdt)
    la.router *= 1 / la.size
    x = la.x(m, xdt)
    resid = torch.randn(m, la.k, generator=la.gen).to(ydt).to(dev)
    bias = (0.1 * torch.randn(9, generator=la.gen)).to(dev)
    y, ids, w = run(la, x, 3, act=1, score=1, renorm=False, scale=2.5, router_bias=bias, resid=resid, out_dtype=ydt, save=True)
    assert y.dtype == ydt and ids.dtype == torch.int32 and w.dtype == torch.float32
    rid, rw = choose(x, la.router, 3, 1, False, 2.5, bias)
    assert torch.equal(ids.long(), rid)
    check(la, x, rid, rw, 1, resid, y)


@pytest.mark.parametrize("m", [1, 3, 4, 5, 33])
@pytest.mark.parametrize("dtype", DTYPES)
def test_nothing_behind_the_outputs(dev, m, dtype):
    """Values before and behind the outputs stay as they were, at any alignment of the operands."""
    import gq
    la = Layer(dev, O.Q4_0, O.Q8_0, 5, 96, 288, seed=6, router=dtype)
    la.router *= 1 / la.size
    x0, top = la.x(m, dtype), 3
    resid0 = torch.randn(m, la.k, generator=la.gen).to(dtype).to(dev)

    def guarded(rows, cols, at, dt=dtype):
        buf = torch.full((at + rows * cols + 2000,), 7, dtype=dt, device=dev)
        return buf, buf[at:at + rows * cols].view(rows, cols)

    for at in (0, 1, 3):
        (yb, y), (ib, ids), (wb, w) = guarded(m, la.k, at), guarded(m, top, at, torch.int32), guarded(m, top, at, torch.float32)
        x, resid = guarded(m, la.k, at)[1].copy_(x0), guarded(m, la.k, at)[1].copy_(resid0)
        router = guarded(la.e, la.k, at)[1].copy_(la.router)
        gq.moe_layer(la.fmt, *la.packed[:2], la.fmt_down, la.packed[2], router, x, la.n, la.k, la.e, top, resid=resid, y=y, ids=ids, weights=w)
        rid, rw = choose(x, router, top, 0, True, 1.0, None)
        assert torch.equal(ids.long(), rid)
        check(la, x, rid, rw, 0, resid, y)
        first = y.clone()
        y.fill_(7)
        products(la, x, ids, w, resid=resid, y=y)
        assert torch.equal(y, first)
        ids.fill_(7)
        w.fill_(7)
        gq.moe_route(router, x, la.k, la.e, top, ids=ids, weights=w)
        assert torch.equal(ids.long(), rid)
        for buf, o in ((yb, y), (ib, ids), (wb, w)):
            assert bool((buf[:at] == 7).all()) and bool((buf[at + o.numel():] == 7).all())


@pytest.mark.parametrize("m", [1, 4, 16, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sizes_of_rows(dev, m, dtype):
    """Tokens far outside fp16's range, in both directions, keep their precision (h of twice the power)."""
    la = Layer(dev, O.Q8_0, O.Q8_0, 4, 128, 512, seed=7)
    s = torch.exp2(torch.randint(-30, 30, (m, 1), generator=la.gen).double()).to(dev)
    x = (la.x(m, dtype).double() * s).to(dtype)
    ids, w = random_choice(la, m, 2)
    check(la, x, ids.long(), w, 0, None, products(la, x, ids, w, out_dtype=torch.float32))


def test_closed_gates(dev):
    """Gates so low that h is zero or below fp16's range in whole blocks: finite outputs, zeros where all of h is zero."""
    e, n, k = 2, 256, 256
    la = Layer(dev, O.Q8_0, O.Q8_0, e, n, k, seed=8)
    for m in (1, 4, 9):
        ids, w = random_choice(la, m, 1)
        for size in (0.0, 30.0, 300.0, 1e5):
            x = (la.x(m, torch.float32) * size)
            y = products(la, x, ids, w)
            check(la, x, ids.long(), w, 0, None, y)
            assert size > 0 or bool((y == 0).all())


def test_streams_and_workspaces(dev):
    """Calls that overlap on two streams, with workspaces of their own and without."""
    import gq
    la = Layer(dev, O.Q4_K, O.Q4_K, 8, 512, 1024, seed=9)
    la.router *= 1 / la.size
    xs = [la.x(m, torch.bfloat16) for m in (1, 4, 12, 64)]
    ref = [run(la, x, 2, save=True) for x in xs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    ws = [gq.Workspace(dev) for _ in range(2)]
    outs = []
    for i in range(16):
        s, j = i % 2, (i // 2) % 4
        with torch.cuda.stream(streams[s]):
            outs.append((j, run(la, xs[j], 2, save=True, workspace=ws[s] if i < 8 else None)))
    torch.cuda.synchronize()
    for j, got in outs:
        assert all(torch.equal(a, b) for a, b in zip(got, ref[j]))


@pytest.mark.parametrize("m", [1, 3, 12, 64])
def test_captured(dev, m):
    """The router, the products and the layer in a graph, replayed on new tokens with eager work between the replays."""
    import gq
    e, top = 40, 4
    la = Layer(dev, O.Q4_K, O.Q6_K, e, 256, 512, seed=10)
    la.router *= 1 / la.size
    x = la.x(m, torch.bfloat16)
    ws = gq.Workspace(dev, gq.moe_workspace_bytes(la.fmt, la.fmt_down, m, la.n, la.k, e, top) + 8 * m * e)
    y, y2 = torch.empty_like(x), torch.empty_like(x)
    ids, ids2 = (torch.empty(m, top, dtype=torch.int32, device=dev) for _ in range(2))
    w, w2 = torch.empty(m, top, device=dev), torch.empty(m, top, device=dev)
    every = (y, y2, w, w2, ids, ids2)

    def step():
        run(la, x, top, y=y, ids=ids, weights=w, workspace=ws)
        gq.moe_route(la.router, x, la.k, e, top, ids=ids2, weights=w2, workspace=ws)
        products(la, x, ids2, w2, y=y2, workspace=ws)

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for i in range(4):
        x.copy_(la.x(m, torch.bfloat16))
        for t in every:
            t.fill_(-5)
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in every]
        step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, every))
        assert torch.equal(y, y2) and torch.equal(ids, ids2) and torch.equal(w, w2)
        rid, rw = choose(x, la.router, top, 0, True, 1.0, None)
        assert torch.equal(ids.long(), rid)
        check(la, x, rid, rw, 0, None, y)


def test_repeatable(dev):
    la = Layer(dev, O.Q4_0, O.Q4_0, 16, 1024, 2048, seed=11)
    la.router *= 1 / la.size
    for m in (1, 4, 7, 64):
        x = la.x(m, torch.bfloat16)
        first = run(la, x, 8, save=True)
        for _ in range(3):
            assert all(torch.equal(a, b) for a, b in zip(run(la, x, 8, save=True), first))


@pytest.mark.parametrize("e,top,n,k", [(8, 2, 256, 512), (40, 8, 96, 2048), (3, 3, 64, 17024)])
def test_a_workspace_for_more_tokens_serves_fewer(dev, e, top, n, k):
    """The bytes given for 64 tokens are taken for every call of fewer, one byte less is refused, and nothing is written behind them."""
    import ctypes

    import gq
    la, lib = Layer(dev, O.Q4_0, O.Q8_0, e, n, k, seed=12) if n % 256 else Layer(dev, O.Q4_K, O.Q6_K, e, n, k, seed=12), gq.load()
    s = torch.cuda.current_stream().cuda_stream
    x64 = la.x(64, torch.float32)
    for m in (1, 2, 4, 5, 16, 17, 63, 64):
        x, (ids, w) = x64[:m], random_choice(la, m, top, m)
        layer = gq.MoeLayer(la.fmt, la.fmt_down, 0, top, *(p.data_ptr() for p in la.packed), e, n, k, la.router.data_ptr(), None, gq.DT_F32, 0, 1, 1.0)
        at, own = ctypes.addressof(layer), gq.moe_workspace_bytes(la.fmt, la.fmt_down, m, n, k, e, top)
        need = gq.moe_workspace_bytes(la.fmt, la.fmt_down, 64, n, k, e, top)
        buf, y = torch.full((need + 65536,), 7, dtype=torch.uint8, device=dev), torch.empty(m, k, device=dev)
        for nbytes, status in ((own - 1, 4), (own, 0), (need, 0)):
            y.fill_(NAN)
            assert lib.gq_moe_ffn(at, x.data_ptr(), gq.DT_F32, ids.data_ptr(), w.data_ptr(), None, y.data_ptr(), gq.DT_F32, m, buf.data_ptr(),
                                  nbytes, s) == status
            assert bool((buf[max(own, nbytes):] == 7).all())
            if status == 0:
                check(la, x, ids.long(), w, 0, None, y)
        assert lib.gq_moe_layer(at, x.data_ptr(), gq.DT_F32, None, y.data_ptr(), gq.DT_F32, None, None, m, buf.data_ptr(), own - 1, s) == 4
        assert lib.gq_moe_layer(at, x.data_ptr(), gq.DT_F32, None, y.data_ptr(), gq.DT_F32, None, None, m, buf.data_ptr(), own, s) == 0
        rid, rw = choose(x, la.router, top, 0, True, 1.0, None)
        check(la, x, rid, rw, 0, None, y)
        buf.fill_(7)
        room = lib.gq_moe_route_workspace_bytes(at, m)
        assert lib.gq_moe_route(at, x.data_ptr(), gq.DT_F32, ids.data_ptr(), w.data_ptr(), m, buf.data_ptr(), room - 1, s) == 4
        assert lib.gq_moe_route(at, x.data_ptr(), gq.DT_F32, ids.data_ptr(), w.data_ptr(), m, buf.data_ptr(), room, s) == 0
        assert torch.equal(ids.long(), rid) and bool((buf[room:] == 7).all())


def test_empty(dev):
    import gq
    la = Layer(dev, O.Q8_0, O.Q8_0, 4, 32, 64, seed=13)
    x = torch.empty(0, 64, dtype=torch.bfloat16, device=dev)
    y, ids, w = run(la, x, 2, save=True, workspace=gq.Workspace(dev))
    assert y.shape == (0, 64) and ids.shape == w.shape == (0, 2)
    assert products(la, x, ids, w).shape == (0, 64)
    assert gq.moe_route(la.router, x, 64, 4, 2)[0].shape == (0, 2)


def test_capture_without_a_workspace(dev):
    """A call takes no workspace of its own while its stream is captured."""
    import gq
    la = Layer(dev, O.Q8_0, O.Q8_0, 4, 64, 64, seed=14)
    xs, out = [la.x(m, torch.bfloat16) for m in (2, 9)], torch.empty(9, 64, dtype=torch.bfloat16, device=dev)
    choice = [random_choice(la, len(x), 2) for x in xs]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for x, (ids, w) in zip(xs, choice):
            for call in (lambda: run(la, x, 2, y=out[:len(x)], ids=ids, weights=w), lambda: products(la, x, ids, w, y=out[:len(x)]),
                         lambda: gq.moe_route(la.router, x, 64, 4, 2, ids=ids, weights=w)):
                with pytest.raises(gq.GQError):
                    call()
        out.fill_(3)
    graph.replay()
    torch.cuda.synchronize()
    assert bool((out == 3).all())


def test_a_given_stream_owns_the_outputs(dev):
    """Outputs made for a call on another stream do not lie in memory that queued work of the current one still writes."""
    import gq
    la = Layer(dev, O.Q8_0, O.Q8_0, 8, 512, 2048, seed=15)
    la.router *= 1 / la.size
    x = la.x(64, torch.bfloat16)
    ref = run(la, x, 2, save=True)
    side, a = torch.cuda.Stream(), torch.randn(8192, 8192, device=dev).to(torch.bfloat16)
    calls = [(lambda: run(la, x, 2, save=True, stream=side), ref), (lambda: (products(la, x, ref[1], ref[2], stream=side),), ref[:1]),
             (lambda: gq.moe_route(la.router, x, la.k, la.e, 2, stream=side), ref[1:])]
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
        for p, q in zip(got, want):
            assert torch.equal(p, q)


def test_operands_elsewhere_are_refused(dev):
    """A stream of another device, operands of other shapes and types, and no kernel gets the address of host memory."""
    import types

    import gq
    la = Layer(dev, O.Q8_0, O.Q8_0, 4, 64, 64, seed=16)
    x = la.x(9, torch.bfloat16)
    ids, w = random_choice(la, 9, 2)
    far = types.SimpleNamespace(device=torch.device("cuda:7"), cuda_stream=0)
    for call in (lambda **kw: run(la, x, 2, **kw), lambda **kw: products(la, x, ids, w, **kw),
                 lambda **kw: gq.moe_route(la.router, x, 64, 4, 2, **kw)):
        with pytest.raises(gq.GQError, match="cuda:7"):
            call(stream=far)
        with pytest.raises(gq.GQError, match="workspace"):
            call(workspace=gq.Workspace("cpu"))
    for name, bad in (("resid", x.float()), ("resid", x.cpu()), ("y", x[:8]), ("ids", ids.long()), ("ids", ids[:, :1]), ("weights", w.double()),
                      ("router_bias", torch.zeros(4, device=dev).half()), ("router_bias", torch.zeros(5, device=dev))):
        with pytest.raises(gq.GQError, match=name):
            run(la, x, 2, **{name: bad})
    with pytest.raises(gq.GQError, match="ids"):
        products(la, x, ids[:8], w)
    with pytest.raises(gq.GQError, match="ids"):
        products(la, x, ids[0], w)
    with pytest.raises(gq.GQError, match="weights"):
        products(la, x, ids, w.cpu())
    with pytest.raises(gq.GQError, match="router"):
        gq.moe_route(la.router[:3], x, 64, 4, 2)
    for i, name in enumerate(("gate", "up", "down")):
        packed = [p[:-16] if j == i else p for j, p in enumerate(la.packed)]
        with pytest.raises(gq.GQError, match=name):
            gq.moe_ffn(la.fmt, *packed[:2], la.fmt_down, packed[2], x, ids, w, 64, 64, 4)
    with pytest.raises(gq.GQError):  # (more tokens than the layer takes)
        products(la, la.x(65, torch.bfloat16), *random_choice(la, 65, 2))


def test_a_workspace_outgrown_after_a_capture(dev):
    """A captured call's workspace is not given to others when a later call needs a larger one."""
    import gq
    la = Layer(dev, O.Q4_K, O.Q4_K, 8, 512, 512, seed=17)
    la.router *= 1 / la.size
    x, big = la.x(7, torch.bfloat16), la.x(64, torch.bfloat16)
    ws = gq.Workspace(dev, gq.moe_workspace_bytes(la.fmt, la.fmt_down, 7, 512, 512, 8, 2))
    y = torch.empty_like(x)
    run(la, x, 2, y=y, workspace=ws)
    torch.cuda.synchronize()
    ref, graph = y.clone(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        run(la, x, 2, y=y, workspace=ws)
    size = ws.buf.numel()
    run(la, big, 2, workspace=ws)
    assert ws.buf.numel() > size
    torch.cuda.synchronize()
    others = [torch.full((size,), 7, dtype=torch.uint8, device=dev) for _ in range(3)]
    for _ in range(3):
        y.fill_(NAN)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, ref) and all(bool((t == 7).all()) for t in others)


def test_calls_of_several_threads(dev):
    """Threads on streams of their own, without workspaces: each call's result is what it is alone."""
    import threading
    la = Layer(dev, O.Q6_K, O.Q4_0, 8, 256, 1024, seed=18)
    la.router *= 1 / la.size
    xs = [la.x(m, torch.bfloat16) for m in (1, 4, 20, 64)]
    want = [run(la, x, 2, save=True) for x in xs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    if not all(torch.equal(a, b) for a, b in zip(run(la, xs[i], 2, save=True), want[i])):
                        wrong.append(i)
        except Exception as e:  # (a thread's exception would be lost)
            wrong.append(repr(e))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(xs))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_two_captured_graphs_replayed_together(dev):
    """Two graphs with workspaces of their own, replayed at once on two streams."""
    import gq
    la = Layer(dev, O.Q4_0, O.Q4_0, 8, 1024, 2048, seed=19)
    la.router *= 1 / la.size
    made = []
    for m in (4, 40):
        x, ws = la.x(m, torch.bfloat16), gq.Workspace(dev)
        y = torch.empty_like(x)
        run(la, x, 2, y=y, workspace=ws)
        torch.cuda.synchronize()
        want, graph = y.clone(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            run(la, x, 2, y=y, workspace=ws)
        made.append((graph, torch.cuda.Stream(), y, want, x, ws))
    for _ in range(4):
        for made_one in made:
            made_one[2].fill_(NAN)
        torch.cuda.synchronize()
        for graph, stream, *_ in made:
            with torch.cuda.stream(stream):
                for _ in range(5):
                    graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(y, want) for _, _, y, want, *_ in made)


@pytest.mark.parametrize("m", [2, 9])
def test_expert_tensors_past_4_gib(dev, m):
    """120 experts of 4096 x 20480 at 4.5 bits: 5.7 GB a tensor."""
    import gq
    fmt, e, n, k, top = O.Q4_0, 120, 4096, 20480, 2
    gen = torch.Generator(device="cuda").manual_seed(5)
    packed, picked, w = [], [0, 60, 90, 119], []
    for rows, cols in ((n, k), (n, k), (k, n)):
        b = torch.randint(0, 256, (e * rows * cols // 32, 18), generator=gen, device=dev, dtype=torch.uint8)
        b[:, 0], b[:, 1] = 0, 0x24  # (scales of 2^-6)
        part = b.view(e, -1)[picked].cpu().numpy()
        w.append({i: torch.from_numpy(O.dequant(fmt, np.ascontiguousarray(p)).reshape(rows, cols)).to(dev).double() for i, p in zip(picked, part)})
        packed.append(gq.repack(fmt, b.view(-1), e * rows, cols))
        del b
    x = (torch.randn(m, k, generator=torch.Generator().manual_seed(6)) * 0.05).to(torch.bfloat16).to(dev)
    ids = torch.tensor([[picked[i % 4], picked[(i + 1) % 4]] for i in range(m)], dtype=torch.int32, device=dev)
    wt = torch.rand(m, top, generator=torch.Generator().manual_seed(7)).to(dev)
    y = gq.moe_ffn(fmt, packed[0], packed[1], fmt, packed[2], x, ids, wt, n, k, e)
    la = Layer.__new__(Layer)
    la.e, la.n, la.k, la.w = e, n, k, w
    check(la, x, ids.long(), wt, 0, None, y)


def test_a_tensor_of_a_file(dev, tmp_path):
    """A GGUF file's three-dimensional expert tensors load as the rows of all experts, one behind the other."""
    import gq
    from gguf_writer import GGML_Q4_0, GGML_Q8_0, llama_kv, write_gguf
    e, n, k, m = 5, 64, 96, 6
    raws = [O.gen_weights(f, e * rows, cols, seed=i) for i, (f, rows, cols) in enumerate(((O.Q4_0, n, k), (O.Q4_0, n, k), (O.Q8_0, k, n)))]
    path = str(tmp_path / "moe.gguf")
    write_gguf(path, llama_kv(), [("blk.0.ffn_gate_exps.weight", [k, n, e], GGML_Q4_0, raws[0].tobytes()),
                                  ("blk.0.ffn_up_exps.weight", [k, n, e], GGML_Q4_0, raws[1].tobytes()),
                                  ("blk.0.ffn_down_exps.weight", [n, k, e], GGML_Q8_0, raws[2].tobytes())])
    la = Layer.__new__(Layer)
    la.dev, la.e, la.n, la.k, la.fmt, la.fmt_down = dev, e, n, k, O.Q4_0, O.Q8_0
    la.w = [torch.from_numpy(O.dequant(f, b).reshape(e, rows, cols)).to(dev).double() for b, (f, rows, cols) in
            zip(raws, ((O.Q4_0, n, k), (O.Q4_0, n, k), (O.Q8_0, k, n)))]
    with gq.GGUF(path) as g:
        loaded = [g.load(f"blk.0.ffn_{name}_exps.weight", gq.LOAD_QUANT, device=dev) for name in ("gate", "up", "down")]
    la.packed = [t[0] for t in loaded]
    assert [(t[3]["fmt"], t[3]["N"], t[3]["K"]) for t in loaded] == [(O.Q4_0, e * n, k), (O.Q4_0, e * n, k), (O.Q8_0, e * k, n)]
    x = (torch.randn(m, k, generator=torch.Generator().manual_seed(1)) * 0.3).to(torch.bfloat16).to(dev)
    ids, w = random_choice(la, m, 3)
    check(la, x, ids.long(), w, 0, None, products(la, x, ids, w))


@pytest.mark.parametrize("fmt,down", [(O.Q4_K, O.Q6_K), (O.Q8_0, O.Q4_0)])
def test_a_block_decodes(dev, fmt, down):
    """The operators as they are used together: projections with a bias, a projection added to the stream in place, and the experts
    added to it; a step of many sequences agrees with each sequence by itself."""
    import gq
    from test_gpu_linear import Case, check_forward
    m, n, k, e, top = 24, 256, 512, 12, 3
    la = Layer(dev, fmt, down, e, n, k, seed=20)
    qkv, out = Case(dev, fmt, m, k + 256, k, seed=21, resid=False), Case(dev, down, m, k, k, seed=22, bias=False, resid=False)
    gen = torch.Generator().manual_seed(3)
    stream = torch.randn(m, k, generator=gen).to(torch.bfloat16).to(dev)
    ws = gq.Workspace(dev)

    def block(x, stream):
        """(the attention between the projections is left out: its values are the projection's)"""
        z = gq.linear(fmt, qkv.packed, x, k + 256, k, bias=qkv.bias, workspace=ws)
        a = z[:, :k].contiguous()
        s = gq.linear(down, out.packed, a, k, k, resid=stream, y=stream.clone(), workspace=ws)
        t = (s.float() * la.size).to(torch.bfloat16)
        y, ids, w = run(la, t, top, resid=s, save=True, workspace=ws)
        return z, a, s, t, y, ids, w

    la.router *= 1 / la.size
    z, a, s, t, y, ids, w = block(qkv.x, stream)
    check_forward(qkv, gq.ACT_NONE, z, None, torch.bfloat16)
    out.x, out.resid = a, stream
    check_forward(out, gq.ACT_NONE, s, None, torch.bfloat16)
    rid, rw = choose(t, la.router, top, 0, True, 1.0, None)
    assert torch.equal(ids.long(), rid)
    check(la, t, rid, rw, 0, s, y)
    for i in (0, 11, 23):
        one = run(la, t[i:i + 1], top, resid=s[i:i + 1], save=True, workspace=ws)
        assert torch.equal(one[1], ids[i:i + 1]) and torch.equal(one[2], w[i:i + 1])
        check(la, t[i:i + 1], rid[i:i + 1], rw[i:i + 1], 0, s[i:i + 1], one[0])


@pytest.mark.parametrize("m", [1, 3, 9, 64])
def test_no_expert_at_all(dev, m):
    """Ids that all name none: the residual, or zeros."""
    la = Layer(dev, O.Q4_K, O.Q8_0, 3, 256, 256, seed=25)
    x, w = la.x(m, torch.bfloat16), torch.rand(m, 2, generator=la.gen).to(dev)
    ids = torch.full((m, 2), -1, dtype=torch.int32, device=dev)
    ids[:, 1] = 3
    resid = torch.randn(m, 256, generator=la.gen).to(torch.bfloat16).to(dev)
    assert bool((products(la, x, ids, w) == 0).all())
    assert torch.equal(products(la, x, ids, w, resid=resid), resid)


@pytest.mark.parametrize("m,e,top", [(64, 1024, 16), (64, 16, 16), (4, 1024, 16)])
def test_the_most(dev, m, e, top):
    """As many tokens, experts and experts a token as a call takes."""
    la = Layer(dev, O.Q4_0, O.Q8_0, e, 32, 64, seed=26)
    la.router *= 1 / la.size
    x = la.x(m, torch.float16)
    y, ids, w = run(la, x, top, save=True)
    rid, rw = choose(x, la.router, top, 0, True, 1.0, None)
    assert torch.equal(ids.long(), rid)
    check(la, x, rid, rw, 0, None, y)


@pytest.mark.parametrize("m", [2, 7, 40])
def test_half_of_the_choice_wanted(dev, m):
    """ids or weights alone, through the C entry point; y in place of the residual."""
    import ctypes

    import gq
    la, lib = Layer(dev, O.Q8_0, O.Q8_0, 9, 64, 96, seed=27), gq.load()
    la.router *= 1 / la.size
    x = la.x(m, torch.bfloat16)
    resid = torch.randn(m, 96, generator=la.gen).to(torch.bfloat16).to(dev)
    y, ids, w = run(la, x, 3, resid=resid, save=True)
    layer = gq.MoeLayer(la.fmt, la.fmt_down, 0, 3, *(p.data_ptr() for p in la.packed), 9, 64, 96, la.router.data_ptr(), None, gq.DT_F32, 0, 1, 1.0)
    for ids2, w2 in ((torch.empty_like(ids), None), (None, torch.empty_like(w)), (None, None)):
        out = resid.clone()
        st = lib.gq_moe_layer(ctypes.addressof(layer), x.data_ptr(), gq.DT_BF16, out.data_ptr(), out.data_ptr(), gq.DT_BF16,
                              ids2.data_ptr() if ids2 is not None else None, w2.data_ptr() if w2 is not None else None, m, None, 0,
                              torch.cuda.current_stream().cuda_stream)
        assert st == 0 and torch.equal(out, y)
        assert ids2 is None or torch.equal(ids2, ids)
        assert w2 is None or torch.equal(w2, w)
