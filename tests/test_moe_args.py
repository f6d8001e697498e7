"""CPU tests of the mixture-of-experts layer: what the C entry points and the binding refuse, empty calls, sizes.  No pointer here is
read."""
import ctypes

import pytest
import torch

import gq

P = 4096  # a non-null address that no refused or empty call touches
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 4
BIG = (1 << 24) + 32
FIELDS = dict(fmt=gq.FMT_Q4_0, fmt_down=gq.FMT_Q8_0, act=gq.ACT_SILU, top_k=2, gate=P, up=P, down=P, n_experts=8, N=64, K=256, router=P,
              router_bias=None, router_dtype=gq.DT_F32, score=gq.SCORE_SOFTMAX, renorm=1, scale=1.0)


def layer(**kw):
    unknown = set(kw) - set(FIELDS)
    assert not unknown, unknown
    return gq.MoeLayer(*(dict(FIELDS, **kw).values()))



def route(l=True, x=P, xdt=gq.DT_BF16, ids=P, weights=P, m=3, ws=None, ws_bytes=0, **kw):
    s = layer(**kw)
    return gq.load().gq_moe_route(ctypes.addressof(s) if l else None, x, xdt, ids, weights, m, ws, ws_bytes, None)


def ffn(l=True, x=P, xdt=gq.DT_BF16, ids=P, weights=P, resid=None, y=P, dt=gq.DT_BF16, m=3, ws=None, ws_bytes=0, **kw):
    s = layer(**kw)
    return gq.load().gq_moe_ffn(ctypes.addressof(s) if l else None, x, xdt, ids, weights, resid, y, dt, m, ws, ws_bytes, None)


def both(l=True, x=P, xdt=gq.DT_BF16, resid=None, y=P, dt=gq.DT_BF16, ids=None, weights=None, m=3, ws=None, ws_bytes=0, **kw):
    s = layer(**kw)
    return gq.load().gq_moe_layer(ctypes.addressof(s) if l else None, x, xdt, resid, y, dt, ids, weights, m, ws, ws_bytes, None)


EVERY = [(dict(l=False), INVALID), (dict(m=65), UNSUPPORTED), (dict(n_experts=1025), UNSUPPORTED), (dict(top_k=0), UNSUPPORTED),
         (dict(top_k=17, n_experts=64), UNSUPPORTED), (dict(top_k=-1), UNSUPPORTED), (dict(n_experts=0), INVALID), (dict(K=0), INVALID),
         (dict(K=BIG), INVALID), (dict(xdt=3), UNSUPPORTED), (dict(xdt=-1), UNSUPPORTED), (dict(x=None), INVALID),
         (dict(ws=P, ws_bytes=64), WORKSPACE), (dict(ws=P + 8, ws_bytes=1 << 40), INVALID)]
ROUTER = [(dict(router=None), INVALID), (dict(router_dtype=3), UNSUPPORTED), (dict(score=2), UNSUPPORTED), (dict(score=-1), UNSUPPORTED),
          (dict(top_k=9), INVALID)]
PRODUCTS = [(dict(fmt=3), UNSUPPORTED), (dict(fmt=gq.FMT_F16), UNSUPPORTED), (dict(fmt_down=gq.FMT_F16), UNSUPPORTED), (dict(act=2), UNSUPPORTED), (dict(act=-1), UNSUPPORTED),
            (dict(N=0), INVALID), (dict(N=BIG), INVALID), (dict(K=264), INVALID), (dict(N=72), INVALID), (dict(fmt=gq.FMT_Q4_K, K=128), INVALID),
            (dict(fmt_down=gq.FMT_Q6_K, N=128), INVALID), (dict(gate=None), INVALID), (dict(up=None), INVALID), (dict(down=None), INVALID),
            (dict(gate=P + 8), INVALID), (dict(up=P + 4), INVALID), (dict(down=P + 2), INVALID), (dict(y=None), INVALID),
            (dict(dt=3), UNSUPPORTED), (dict(n_experts=1024, N=1 << 15), INVALID)]  # (2^25 rows)


@pytest.mark.parametrize("call", [route, ffn, both])
@pytest.mark.parametrize("bad,status", EVERY)
def test_every_call_refuses(call, bad, status):
    assert call(**bad) == status


@pytest.mark.parametrize("call", [route, both])
@pytest.mark.parametrize("bad,status", ROUTER)
def test_the_router_refuses(call, bad, status):
    assert call(**bad) == status


@pytest.mark.parametrize("call", [ffn, both])
@pytest.mark.parametrize("bad,status", PRODUCTS)
def test_the_products_refuse(call, bad, status):
    assert call(**bad) == status


def test_refuse_their_own():
    assert route(K=260) == INVALID  # (whole 8s)
    assert route(ids=None) == INVALID and route(weights=None) == INVALID
    assert ffn(ids=None) == INVALID and ffn(weights=None) == INVALID


def test_empty_calls():
    assert route(m=0, x=None, ids=None, weights=None, router=None) == OK
    assert ffn(m=0, x=None, y=None, gate=None, up=None, down=None) == OK and both(m=0, x=None, y=None, router=None) == OK
    size = gq.load().gq_moe_workspace_bytes
    for bad, m in ((dict(), 0), (dict(), 65), (dict(fmt=3), 1), (dict(top_k=17), 1), (dict(N=0), 1)):
        s = layer(**bad)
        assert size(ctypes.addressof(s), m) == 0
    assert size(None, 1) == 0 and gq.load().gq_moe_route_workspace_bytes(None, 1) == 0
    s = layer()
    assert gq.load().gq_moe_route_workspace_bytes(ctypes.addressof(s), 0) == 0
    assert gq.load().gq_moe_route_workspace_bytes(ctypes.addressof(s), 5) == 5 * 8 * 8


@pytest.mark.parametrize("e,top,n,k", [(1, 1, 32, 32), (8, 2, 14336, 4096), (64, 8, 1024, 2048), (1024, 16, 64, 256), (16, 16, 4096, 20480),
                                       (3, 2, 32768, 64), (5, 5, 256, 40960)])
def test_workspace_grows_with_the_tokens(e, top, n, k):
    """What suffices for M tokens suffices for fewer."""
    sizes = [gq.moe_workspace_bytes(gq.FMT_Q4_0, gq.FMT_Q8_0, m, n, k, e, top) for m in range(1, 65)]
    assert sizes[0] > 0 and all(a <= b for a, b in zip(sizes, sizes[1:]))


def test_binding_refuses_host_tensors():
    x, w = torch.zeros(4, 256, dtype=torch.bfloat16), torch.zeros(gq.packed_size(gq.FMT_Q4_0, 8 * 64, 256), dtype=torch.uint8)
    d = torch.zeros(gq.packed_size(gq.FMT_Q4_0, 8 * 256, 64), dtype=torch.uint8)
    r, ids, weights = torch.zeros(8, 256), torch.zeros(4, 2, dtype=torch.int32), torch.zeros(4, 2)
    with pytest.raises(gq.GQError):
        gq.moe_route(r, x, 256, 8, 2)
    with pytest.raises(gq.GQError):
        gq.moe_ffn(gq.FMT_Q4_0, w, w, gq.FMT_Q4_0, d, x, ids, weights, 64, 256, 8)
    with pytest.raises(gq.GQError):
        gq.moe_layer(gq.FMT_Q4_0, w, w, gq.FMT_Q4_0, d, r, x, 64, 256, 8, 2)
