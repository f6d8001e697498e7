"""CPU tests of the product with its epilogue: what the C entry points and the binding refuse, empty calls, sizes, and the
gradient formulas against differences.  No pointer here is read."""
import pytest
import torch

import gq
from linear_ref import act_grad

P = 4096  # a non-null address that no refused or empty call touches
OK, INVALID, UNSUPPORTED, WORKSPACE = 0, 1, 2, 4
BIG = (1 << 24) + 32
ACTS = [gq.ACT_SILU, gq.ACT_GELU_TANH, gq.ACT_NONE, gq.ACT_RELU]


def linear(fmt=gq.FMT_Q4_0, w=P, x=P, xdt=gq.DT_BF16, bias=None, bdt=gq.DT_F32, act=gq.ACT_NONE, resid=None, y=P, dt=gq.DT_BF16,
           z=None, m=8, n=64, k=256, ws=None, ws_bytes=0):
    return gq.load().gq_linear(fmt, w, x, xdt, bias, bdt, act, resid, y, dt, z, m, n, k, ws, ws_bytes, None)


def bwd(fmt=gq.FMT_Q4_0, w=P, dy=P, z=P, dt=gq.DT_BF16, act=gq.ACT_RELU, dz=P, dx=P, xdt=gq.DT_BF16, dbias=P, m=8, n=64,
        k=256, ws=None, ws_bytes=0):
    return gq.load().gq_linear_bwd(fmt, w, dy, z, dt, act, dz, dx, xdt, dbias, m, n, k, ws, ws_bytes, None)


@pytest.mark.parametrize("call", [linear, bwd])
@pytest.mark.parametrize("bad,status", [
    (dict(fmt=3), UNSUPPORTED), (dict(fmt=gq.FMT_F16), UNSUPPORTED), (dict(act=4), UNSUPPORTED), (dict(act=-1), UNSUPPORTED),
    (dict(xdt=3), UNSUPPORTED), (dict(dt=-1), UNSUPPORTED), (dict(k=33), INVALID), (dict(fmt=gq.FMT_Q4_K, k=128), INVALID),
    (dict(n=BIG), INVALID), (dict(k=BIG), INVALID), (dict(m=BIG), INVALID), (dict(w=None), INVALID), (dict(w=P + 8), INVALID),
    (dict(k=0), INVALID),
    # a packed tensor of 4 GiB and more
    (dict(fmt=gq.FMT_Q8_0, n=1 << 20, k=4096), INVALID),
    # a workspace that is too small, or not 16-byte aligned
    (dict(ws=P, ws_bytes=64), WORKSPACE), (dict(ws=P + 8, ws_bytes=1 << 40), INVALID),
])
def test_linear_refuses(call, bad, status):
    assert call(**bad) == status


def test_linear_refuses_its_own():
    assert linear(x=None) == INVALID and linear(y=None) == INVALID
    assert linear(bias=P, bdt=3) == UNSUPPORTED
    assert linear(n=1 << 21, k=32, dt=gq.DT_F32) == INVALID  # (offsets of a tile's outputs)
    assert bwd(dy=None) == INVALID and bwd(z=None) == INVALID


def test_empty_calls():
    assert linear(m=0) == OK and linear(n=0) == OK and linear(m=0, x=None, y=None) == OK and linear(n=0, w=None, y=None) == OK
    assert bwd(m=0, dbias=None) == OK and bwd(m=0, n=0) == OK and bwd(dz=None, dx=None, dbias=None) == OK
    assert bwd(n=0, dx=None) == OK and bwd(n=0, w=None, dy=None, z=None, dx=None) == OK
    for size in (gq.linear_workspace_bytes, gq.linear_bwd_workspace_bytes):
        assert size(gq.FMT_Q4_0, 5, 64, 0) == 0 and size(3, 5, 64, 256) == 0 and size(gq.FMT_Q4_0, BIG, 64, 256) == 0
        assert size(gq.FMT_Q4_0, 5, 64, 256) > 0
    assert gq.linear_bwd_workspace_bytes(gq.FMT_Q4_0, 5, 0, 64) == 0


@pytest.mark.parametrize("size", [gq.linear_workspace_bytes, gq.linear_bwd_workspace_bytes])
@pytest.mark.parametrize("n,k", [(1, 256), (64, 256), (1000, 4096), (14336, 4096), (4096, 14336), (1 << 20, 512)])
def test_workspace_grows_with_the_rows(size, n, k):
    """What suffices for M rows suffices for fewer."""
    rows = sorted({1, 4, 5, 16, 17, 31, 32, 33, 64, 65, 100, 127, 128, 129, 200, 255, 256, 257, 500, 1000, 2048, 5000, 70000})
    for fmt in (gq.FMT_Q4_0, gq.FMT_Q6_K):
        sizes = [size(fmt, m, n, k) for m in rows]
        assert all(a <= b for a, b in zip(sizes, sizes[1:]))


def test_binding_refuses_host_tensors():
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    with pytest.raises(gq.GQError):
        gq.linear(gq.FMT_Q4_0, torch.zeros(gq.packed_size(gq.FMT_Q4_0, 64, 256), dtype=torch.uint8), x, 64, 256)
    with pytest.raises(gq.GQError):
        gq.linear_bwd(gq.FMT_Q4_0, torch.zeros(1, dtype=torch.uint8), x, None, 256, 64)


@pytest.mark.parametrize("act", ACTS)
def test_gradient_formula(act):
    """act' against central differences (their error: h^2 / 6 of the third derivative, below 3, and 2^-53 / h)."""
    z = torch.linspace(-9, 9, 4001, dtype=torch.float64) + 1e-3
    h = 1e-5
    d = (act_grad(act, z + h)[0] - act_grad(act, z - h)[0]) / (2 * h)
    assert float((act_grad(act, z)[1] - d).abs().max()) <= 3 * h * h + 9 * 2 ** -52 / h
