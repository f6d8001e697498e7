"""The gated front and the 4-bit products where a tensor passes 4 GiB, and rows of 16-bit x with an Inf or NaN.

Tolerances are those of test_gpu_ffn and test_gpu_w4."""
import pytest
import torch

import oracle as O
import test_gpu_w4 as W4
from test_gpu_ffn import Case, check_front, check_grads

pytestmark = pytest.mark.gpu
FAR = [0, 1, 70000, 131071, 131072, 149870, 149999]  # rows on both sides of 4 GiB of outputs, and the last


def rows_of(c, rows):
    """The case as if it had these rows alone."""
    r = Case.__new__(Case)
    r.w, r.x, r.g, r.u, r.dh = c.w, c.x[rows], c.g[rows], c.u[rows], c.dh[rows]
    return r


def test_front_and_backward_past_4_gib(dev):
    """150000 x 16384 outputs of 2 bytes: 4.9 GB each."""
    import gq
    fmt, m, n, k = O.Q4_0, 150000, 16384, 64
    c = Case(dev, fmt, 1000, n, k, seed=3)
    c.x = torch.randn(m, k, generator=torch.Generator().manual_seed(4)).to(dev).to(torch.bfloat16) * c.x.abs().mean()
    c.g, c.u, c.dh = (t.repeat(150, 1) for t in (c.g, c.u, c.dh))
    h, g, u = gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, save=True)
    f = rows_of(c, FAR)
    check_front(f, 0, (h[FAR], g[FAR], u[FAR]), torch.bfloat16)
    del h, g, u
    out = gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k)
    check_grads(f, 0, {name: t[FAR] for name, t in out.items()}, torch.bfloat16)


@pytest.mark.parametrize("m", [1, 7])
def test_w4_past_4_gib(dev, m):
    """600000 x 16384 codes: 4.9 GB, and as much again before they are laid out."""
    import gq
    n, k, group = 600000, 16384, 128
    gen = torch.Generator(device="cuda").manual_seed(5)
    q = torch.randint(0, 256, (n, k // 2), generator=gen, device=dev, dtype=torch.uint8)
    s = (0.004 + 0.004 * torch.rand(n, k // group, generator=gen, device=dev)).to(torch.float16)
    z = torch.randint(0, 17, (n, k // group), generator=gen, device=dev, dtype=torch.uint8)
    p = gq.w4_pack(q, s, z, n, k, group)
    x = W4.make_x(dev, m, k, torch.bfloat16, 1)
    y, h = gq.w4_gemv(p, group, x, n, k), gq.w4_gate_up(p, p, group, x, n, k)
    for r in (slice(0, 40), slice(524280, 524320), slice(n - 40, n)):
        codes = torch.stack([q[r] & 15, q[r] >> 4], 2).reshape(40, k).double()
        e = torch.arange(k, device=dev) // group
        ref = x.double() @ (s[r].double()[:, e] * (codes - z[r].double()[:, e])).t().contiguous()
        W4.check(y[:, r], ref)
        W4.check(h[:, r], W4.act_grad(0, ref)[0] * ref, extra=8.0)


@pytest.mark.parametrize("fmt", [O.Q4_0, O.Q8_0, O.Q4_K, O.Q6_K])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("m,k", [(1, 512), (4, 1280), (2, 4096), (3, 4608), (11, 2304), (7, 4352), (24, 2304)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_nonfinite_rows_of_16_bits(dev, fmt, dtype, m, k, bad):
    """Such a row comes out non-finite, the others as without it."""
    import gq
    n = 200
    c = Case(dev, fmt, m, n, k, seed=13, dtype=dtype)
    ref = gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, save=True)
    c.x[m // 2, 100] = bad
    got = gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, save=True)
    keep = [i for i in range(m) if i != m // 2]
    for a, b in zip(got, ref):
        assert not bool(a[m // 2].isfinite().any())
        assert torch.equal(a[keep], b[keep])


@pytest.mark.parametrize("most,n,k", [(65, 2048, 512), (300, 1000, 1024), (96, 520, 4352)])
def test_a_workspace_for_more_rows_serves_fewer(dev, most, n, k):
    """The bytes given for `most` rows are taken for every call of fewer, and nothing is written behind them."""
    import gq
    fmt, lib = O.Q4_0, gq.load()
    c = Case(dev, fmt, most, n, k, seed=7)
    for backward, need in ((False, gq.ffn_gate_up_workspace_bytes(fmt, most, n, k)),
                           (True, gq.ffn_gate_up_bwd_workspace_bytes(fmt, most, n, k))):
        buf = torch.full((need + 65536,), 7, dtype=torch.uint8, device=dev)
        for m in sorted({1, 4, 5, 17, 31, 32, 33, 63, 64, most - 1, most} & set(range(1, most + 1))):
            out, f = torch.empty(m, k if backward else n, dtype=torch.bfloat16, device=dev), rows_of(c, slice(0, m))
            s = torch.cuda.current_stream().cuda_stream
            if backward:
                st = lib.gq_ffn_gate_up_bwd(fmt, c.packed[0].data_ptr(), c.packed[1].data_ptr(), c.dh.data_ptr(), c.g.data_ptr(),
                                            c.u.data_ptr(), gq.DT_BF16, None, None, out.data_ptr(), gq.DT_BF16, m, n, k, 0,
                                            buf.data_ptr(), need, s)
                assert st == 0
                check_grads(f, 0, {"dx": out, "dg": None, "du": None}, torch.bfloat16)
            else:
                st = lib.gq_ffn_gate_up(fmt, c.packed[0].data_ptr(), c.packed[1].data_ptr(), c.x.data_ptr(), gq.DT_BF16,
                                        out.data_ptr(), gq.DT_BF16, None, None, m, n, k, 0, buf.data_ptr(), need, s)
                assert st == 0
                check_front(f, 0, (out, None, None), torch.bfloat16)
            assert bool((buf[need:] == 7).all())


def test_calls_of_several_threads(dev):
    """Threads on streams of their own, without workspaces: each call's result is what it is alone."""
    import threading

    import gq
    fmt, n, k = O.Q6_K, 700, 2304
    cases = [Case(dev, fmt, m, n, k, seed=m) for m in (2, 24, 70, 200)]
    want = [(gq.ffn_gate_up(fmt, *c.packed, c.x, n, k), gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k)["dx"]) for c in cases]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(20):
                    c = cases[i]
                    h, dx = gq.ffn_gate_up(fmt, *c.packed, c.x, n, k), gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k)["dx"]
                    if not (torch.equal(h, want[i][0]) and torch.equal(dx, want[i][1])):
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
    fmt, n, k = O.Q4_K, 1024, 2304
    made = []
    for m in (40, 260):
        c, ws = Case(dev, fmt, m, n, k, seed=m), gq.Workspace(dev)
        h, dx = torch.empty(m, n, dtype=torch.bfloat16, device=dev), torch.empty(m, k, dtype=torch.bfloat16, device=dev)

        def step(c=c, ws=ws, h=h, dx=dx):
            gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, h=h, workspace=ws)
            gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k, dx=dx, want_dgu=False, workspace=ws)

        step()
        torch.cuda.synchronize()
        want, graph = (h.clone(), dx.clone()), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            step()
        made.append((graph, torch.cuda.Stream(), (h, dx), want, step))  # (step: what the graph reads stays alive)
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
