"""The mixture-of-experts layer against the formulas in 64 bits.

Tolerances.  Products as in the other tests of this library (under 1e-3 of a row's norm, an error of one size along a row): g and u
of an expert carry 1e-3 of their rows' rms into h as u act'(g) dg + act(g) du, such an error of h and 1e-3 of W_down h's own
norm go into the token's sum with the expert's weight, and a rounding of the output adds finfo.eps / 2.  The choice is
made in 64 bits on both sides and has to be equal; a weight is rounded once to fp32 (2^-24) from a few 64-bit operations."""
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


def choose(x, router, top, score, renorm, scale, bias):
    """ids, weights in 64 bits; a NaN key is the largest, -Inf is never taken."""
    l = x.double() @ router.double().t().contiguous()
    s = torch.softmax(l, 1) if score == 0 else torch.sigmoid(l)
    key = l if bias is None else s + bias.double()
    key = torch.where(torch.isnan(key), torch.inf, key)
    ids = torch.sort(key, dim=1, descending=True, stable=True).indices[:, :top]
    none = key.gather(1, ids) == -torch.inf
    w = torch.where(none, 0.0, s.gather(1, ids))
    if renorm:
        w = w / w.sum(1, keepdim=True)
    return torch.where(none, -1, ids), torch.where(none, 0.0, w) * scale


class Layer:
    def __init__(self, dev, fmt, fmt_down, e, n, k, seed=0, router=torch.float32):
        import gq
        print(f"fmt={fmt} down={fmt_down} e={e} n={n} k={k} seed={seed}", flush=True)
        self.fmt, self.fmt_down, self.e, self.n, self.k = fmt, fmt_down, e, n, k
        self.packed, self.w = [], []
        for i, (f, rows, cols) in enumerate(((fmt, n, k), (fmt, n, k), (fmt_down, k, n))):
            b = O.gen_weights(f, e * rows, cols, seed=8000 + 3 * seed + i)
            self.packed.append(gq.repack(f, torch.from_numpy(b).to(dev), e * rows, cols))
            self.w.append(torch.from_numpy(O.dequant(f, b).reshape(e, rows, cols)).to(dev).double())
        gen = torch.Generator().manual_seed(seed)
        self.router = (torch.randn(e, k, generator=gen) * 1.5 / k ** 0.5).to(router).to(dev)
        self.gen, self.dev = gen, dev
        self.size = 1.5 / (float(self.w[0].pow(2).mean().sqrt()) * k ** 0.5)

    def x(self, m, dtype):
        return (torch.randn(m, self.k, generator=self.gen) * self.size).to(dtype).to(self.dev)

    def logit_x(self, m, dtype):  # (the router sees x too: of size 1 for logits of size 1.5)
        return torch.randn(m, self.k, generator=self.gen).to(dtype).to(self.dev)

    def reference(self, x, ids, weights, act, resid):
        """y and the bound on a row's error, without the output's rounding."""
        x = x.double()
        y = torch.zeros_like(x) if resid is None else resid.double().clone()
        err = torch.zeros(x.shape[0], dtype=torch.float64, device=x.device)
        for e in range(self.e):
            share = torch.where(ids == e, weights.double(), 0.0).sum(1)
            rows = (ids == e).any(1).nonzero()[:, 0]
            if len(rows) == 0:
                continue
            xe = x[rows]
            g, u = xe @ self.w[0][e].t().contiguous(), xe @ self.w[1][e].t().contiguous()
            f, d = act_grad(act, g)
            out = (f * u) @ self.w[2][e].t().contiguous()
            rms = [t.pow(2).mean(1).sqrt() for t in (g, u)]
            dh = PRODUCT * (rms[0] * (u * d).norm(dim=1) + rms[1] * f.norm(dim=1))
            wd = float(self.w[2][e].pow(2).mean().sqrt()) * self.k ** 0.5
            y[rows] += share[rows, None] * out
            err[rows] += share[rows].abs() * (dh * wd * 1.5 + PRODUCT * out.norm(dim=1))
        return y, err


def check(layer, x, ids, weights, act, resid, y):
    ref, err = layer.reference(x, ids, weights, act, resid)
    d = (y.double() - ref).norm(dim=1)
    assert bool((d <= err + half_step(y.dtype) * ref.norm(dim=1) + 1e-30).all()), (d / ref.norm(dim=1)).max()


ROUTES = [(1, 8, 2, 0, True, 1.0, False), (1, 1, 1, 1, False, 2.5, False), (3, 5, 5, 0, False, 1.0, True), (4, 64, 8, 1, True, 2.5, True),
          (5, 65, 3, 0, True, 1.0, False), (16, 128, 16, 0, False, 0.5, False), (37, 61, 5, 1, True, 1.0, True),
          (64, 257, 8, 0, True, 1.0, True), (63, 1024, 16, 1, False, 1.0, True), (64, 3, 2, 0, True, 1.0, False)]


@pytest.mark.parametrize("k", [32, 96, 2048, 4128])
@pytest.mark.parametrize("m,e,top,score,renorm,scale,bias", ROUTES)
def test_route(dev, m, e, top, score, renorm, scale, bias, k):
    import gq
    gen = torch.Generator().manual_seed(m + e + k)
    x = torch.randn(m, k, generator=gen).to(DTYPES[(m + k) % 3]).to(dev)
    router = (torch.randn(e, k, generator=gen) * 1.5 / k ** 0.5).to(DTYPES[(e + k // 32) % 3]).to(dev)
    b = (0.2 * torch.randn(e, generator=gen)).to(dev) if bias else None
    ids, w = gq.moe_route(router, x, k, e, top, score=score, renorm=renorm, scale=scale, router_bias=b)
    rid, rw = choose(x, router, top, score, renorm, scale, b)
    assert torch.equal(ids.long(), rid)
    assert bool(((w.double() - rw).abs() <= (2 ** -24 + 1e-12) * rw.abs() + 2 ** -149).all())


# tokens, experts, taken, n, k: one token to the most, one expert, all taken, sizes of whole 32-blocks
SHAPES = [(1, 8, 2, 256, 256), (1, 1, 1, 512, 256), (2, 4, 4, 256, 512), (3, 16, 5, 256, 256), (4, 5, 3, 512, 512), (5, 4, 2, 256, 256),
          (16, 8, 2, 512, 256), (17, 3, 3, 256, 256), (37, 11, 5, 256, 512), (64, 8, 2, 256, 256), (64, 2, 2, 512, 256),
          (64, 33, 16, 256, 256)]


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,e,top,n,k", SHAPES)
def test_layer(dev, fmt, m, e, top, n, k):
    import gq
    down = FMTS[(FMTS.index(fmt) + m) % 6]
    dtype, act = DTYPES[(m + n // 256) % 3], (m + fmt) % 2
    la = Layer(dev, fmt, down, e, n, k, seed=m)
    x = la.x(m, dtype)
    la.router *= 1 / la.size
    resid = (torch.randn(m, k, generator=la.gen)).to(dtype).to(dev) if m % 2 else None
    y, ids, w = gq.moe_layer(fmt, la.packed[0], la.packed[1], down, la.packed[2], la.router, x, n, k, e, top, act=act, resid=resid,
                             save=True)
    rid, rw = choose(x, la.router, top, 0, True, 1.0, None)
    assert torch.equal(ids.long(), rid)
    check(la, x, rid, rw, act, resid, y)
    # the two calls apart give the same
    ids2, w2 = gq.moe_route(la.router, x, k, e, top)
    assert torch.equal(ids, ids2) and torch.equal(w, w2)
    y2 = gq.moe_ffn(fmt, la.packed[0], la.packed[1], down, la.packed[2], x, ids, w, n, k, e, act=act, resid=resid)
    assert torch.equal(y, y2)


@pytest.mark.parametrize("fmt,down", [(O.Q4_0, O.Q8_0), (O.Q8_0, O.Q4_0)])
@pytest.mark.parametrize("m,e,top,n,k", [(1, 3, 2, 32, 32), (2, 3, 1, 96, 160), (9, 4, 2, 32, 96), (40, 5, 3, 224, 2080)])
def test_short_chunks(dev, fmt, down, m, e, top, n, k):
    import gq
    la = Layer(dev, fmt, down, e, n, k, seed=n)
    x = la.x(m, torch.float16)
    gen = torch.Generator().manual_seed(5)
    ids = torch.stack([torch.randperm(e, generator=gen)[:top] for _ in range(m)]).int().to(dev)
    w = torch.rand(m, top, generator=gen).to(dev)
    y = gq.moe_ffn(fmt, la.packed[0], la.packed[1], down, la.packed[2], x, ids, w, n, k, e)
    check(la, x, ids, w, 0, None, y)


@pytest.mark.parametrize("m", [1, 2, 4, 5, 30, 64])
@pytest.mark.parametrize("dtype", DTYPES)
def test_given_ids(dev, m, dtype):
    """Ids that name no expert, the same expert twice, tokens without any, negative and zero weights."""
    import gq
    e, top, n, k = 6, 4, 256, 256
    la = Layer(dev, O.Q4_K, O.Q6_K, e, n, k, seed=50 + m)
    x = la.x(m, dtype)
    gen = torch.Generator().manual_seed(m)
    ids = torch.randint(-2, e + 3, (m, top), generator=gen)
    if m > 2:
        ids[1] = torch.tensor([-1, e, 2 ** 31 - 1, -2 ** 31])  # (nothing)
        ids[2] = 3                                             # (one expert, four times)
    w = torch.randn(m, top, generator=gen)
    w[:, 0] = 0
    ids, w = ids.int().to(dev), w.float().to(dev)
    resid = torch.randn(m, k, generator=gen).to(dtype).to(dev)
    kept = resid.clone()
    y = gq.moe_ffn(O.Q4_K, la.packed[0], la.packed[1], O.Q6_K, la.packed[2], x, ids, w, n, k, e, resid=resid)
    assert torch.equal(resid, kept)
    check(la, x, ids.long(), w, 0, resid, y)
    if m > 2:
        assert torch.equal(y[1], resid[1])
    into = gq.moe_ffn(O.Q4_K, la.packed[0], la.packed[1], O.Q6_K, la.packed[2], x, ids, w, n, k, e, resid=resid, y=resid)
    assert into is resid and torch.equal(resid, y)
