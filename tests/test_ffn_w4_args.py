"""CPU tests of the gated feed-forward front and the 4-bit group-scaled products: what the C entry points and the
binding refuse, empty calls, sizes, and the gradient formula against differences.  No pointer here is read."""
import ctypes

import pytest
import torch

import gq

P = 4096  # a non-null address that no refused or empty call touches
OK, INVALID, UNSUPPORTED = 0, 1, 2


def front(fmt=gq.FMT_Q4_0, gate=P, up=P, x=P, xdt=gq.DT_BF16, h=P, hdt=gq.DT_BF16, g=None, u=None, m=4, n=64, k=256, act=0):
    return gq.load().gq_ffn_gate_up(fmt, gate, up, x, xdt, h, hdt, g, u, m, n, k, act, None, 0, None)


def bwd(fmt=gq.FMT_Q4_0, gate=P, up=P, dh=P, g=P, u=P, dt=gq.DT_BF16, dg=P, du=P, dx=P, xdt=gq.DT_BF16, m=4, n=64, k=256,
        act=0):
    return gq.load().gq_ffn_gate_up_bwd(fmt, gate, up, dh, g, u, dt, dg, du, dx, xdt, m, n, k, act, None, 0, None)


def w4(w=P, group=128, x=P, xdt=gq.DT_BF16, y=P, ydt=gq.DT_BF16, n=64, k=256, batch=1):
    return gq.load().gq_w4_gemv(w, group, x, xdt, y, ydt, n, k, batch, None)


def w4_front(gate=P, up=P, group=128, x=P, xdt=gq.DT_BF16, h=P, hdt=gq.DT_BF16, n=64, k=256, batch=1, act=0):
    return gq.load().gq_w4_gate_up(gate, up, group, x, xdt, h, hdt, n, k, batch, act, None)


BIG = (1 << 24) + 32


@pytest.mark.parametrize("call", [front, bwd])
@pytest.mark.parametrize("bad,status", [
    (dict(fmt=3), UNSUPPORTED), (dict(fmt=gq.FMT_F16), UNSUPPORTED), (dict(act=2), UNSUPPORTED), (dict(act=-1), UNSUPPORTED),
    (dict(xdt=3), UNSUPPORTED), (dict(k=33), INVALID), (dict(fmt=gq.FMT_Q4_K, k=128), INVALID), (dict(n=BIG), INVALID),
    (dict(k=BIG), INVALID), (dict(m=BIG), INVALID), (dict(gate=None), INVALID), (dict(up=None), INVALID),
    # a packed tensor of 4 GiB and more
    (dict(fmt=gq.FMT_Q8_0, n=1 << 20, k=4096), INVALID),
    # packed tensors that are not 16-byte aligned
    (dict(gate=P + 8), INVALID), (dict(up=P + 1), INVALID),
])
def test_front_refuses(call, bad, status):
    assert call(**bad) == status


def test_front_refuses_its_own():
    assert front(hdt=7) == UNSUPPORTED
    assert front(x=None) == INVALID and front(h=None) == INVALID and front(k=0) == INVALID
    assert front(n=1 << 22, k=32, hdt=gq.DT_F32) == INVALID  # (offsets of a tile's outputs)
    assert bwd(k=0) == INVALID
    assert bwd(dt=7) == UNSUPPORTED
    assert bwd(dh=None) == INVALID and bwd(g=None) == INVALID and bwd(u=None) == INVALID


def test_empty_calls():
    assert front(m=0) == OK and front(n=0) == OK
    assert bwd(m=0) == OK and bwd(n=0, dx=None) == OK and bwd(n=0, gate=None, up=None, dh=None, g=None, u=None, dx=None) == OK
    assert front(m=0, x=None, h=None) == OK and front(n=0, gate=None, up=None, h=None) == OK and bwd(m=0, dh=None, dx=P) == OK
    for size in (gq.ffn_gate_up_workspace_bytes, gq.ffn_gate_up_bwd_workspace_bytes):
        assert size(gq.FMT_Q4_0, 5, 64, 0) == 0
    assert gq.ffn_gate_up_bwd_workspace_bytes(gq.FMT_Q4_0, 5, 0, 64) == 0
    assert bwd(dg=None, du=None, dx=None) == OK  # nothing wanted
    assert w4(n=0) == OK and w4_front(n=0) == OK and w4(n=0, w=None, y=None) == OK


@pytest.mark.parametrize("call", [w4, w4_front])
@pytest.mark.parametrize("bad,status", [
    (dict(group=0), UNSUPPORTED), (dict(group=16), UNSUPPORTED), (dict(group=-32), UNSUPPORTED), (dict(group=256), UNSUPPORTED),
    (dict(batch=0), UNSUPPORTED), (dict(batch=17), UNSUPPORTED), (dict(batch=-1), UNSUPPORTED), (dict(xdt=3), UNSUPPORTED),
    (dict(n=BIG), INVALID), (dict(k=BIG), INVALID), (dict(k=0), INVALID), (dict(x=None), INVALID),
])
def test_w4_refuses(call, bad, status):
    assert call(**bad) == status


def test_w4_refuses_its_own():
    assert w4(w=P + 4) == INVALID and w4_front(up=P + 8) == INVALID and w4_front(gate=P + 1) == INVALID
    assert w4(w=None) == INVALID and w4(y=None) == INVALID and w4(ydt=9) == UNSUPPORTED
    assert w4_front(gate=None) == INVALID and w4_front(up=None) == INVALID and w4_front(h=None) == INVALID
    assert w4_front(act=5) == UNSUPPORTED and w4_front(hdt=9) == UNSUPPORTED
    pack = gq.load().gq_w4_pack
    assert pack(P, P, gq.DT_F32, P, 16, 128, 128, P, None) == UNSUPPORTED  # (fp32 scales would be rounded)
    assert pack(P, P, gq.DT_F16, P, 16, 128, 100, P, None) == UNSUPPORTED
    for i in (0, 1, 7):
        args = [P, P, gq.DT_F16, P, 16, 128, 128, P, None]
        args[i] = None
        assert pack(*args) == INVALID
    assert pack(P, P, gq.DT_F16, P, 16, 128, 128, P + 4, None) == INVALID
    assert pack(P, P, gq.DT_F16, None, 0, 128, 128, P, None) == OK
    size = ctypes.c_size_t(0)
    assert gq.load().gq_w4_packed_size(16, 128, 128, None) == INVALID
    assert gq.load().gq_w4_packed_size(16, 128, 5, ctypes.byref(size)) == UNSUPPORTED


@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("n,k", [(1, 1), (16, 128), (17, 129), (1000, 4090), (0, 128), (16, 0)])
def test_w4_packed_size(n, k, group):
    tiles, chunks = -(-n // 16), -(-k // 128)
    assert gq.w4_packed_size(n, k, group) == tiles * chunks * (1024 + 64 * (128 // group))


@pytest.mark.parametrize("fmt", sorted(set(gq.FORMATS.values())))
def test_workspaces_stop_growing(fmt):
    """Rows are taken in blocks: a workspace grows to a limit, never past it, and never shrinks as M grows."""
    for size in (gq.ffn_gate_up_workspace_bytes, gq.ffn_gate_up_bwd_workspace_bytes):
        at = [size(fmt, m, 14336, 4096) for m in (1, 16, 64, 300, 2048, 20000, 1 << 20)]
        assert at == sorted(at) and at[-1] <= 1 << 30
        assert size(99, 16, 64, 256) == 0 and size(fmt, BIG, 64, 256) == 0


@pytest.mark.parametrize("n,k", [(14336, 4096), (5003, 4096), (520, 130 * 32), (64, 256), (200, 14336), (100000, 64), (4096, 14336)])
def test_a_workspace_of_more_rows_suffices_for_fewer(n, k):
    """What is made for M rows is enough for every call of fewer: no size is below that of a smaller M, one by one up to
    1200 rows and in odd steps beyond."""
    for size in (gq.ffn_gate_up_workspace_bytes, gq.ffn_gate_up_bwd_workspace_bytes):
        at = [size(gq.FMT_Q4_0, m, n, k) for m in [*range(0, 1201), *range(1201, 200000, 997)]]
        assert all(a <= b for a, b in zip(at, at[1:]))


@pytest.mark.parametrize("fmt", sorted(set(gq.FORMATS.values())))
@pytest.mark.parametrize("m", [1, 17, 33, 300, 5000])
def test_scratch_suffices_for_long_rows(fmt, m):
    """Blocks of rows get shorter as the rows get longer: a call without a workspace fits what it may take by itself
    (128 MiB), up to a front's K of 2^21 and any N of a backward pass."""
    for k in (256, 4096, 1 << 17, 1 << 20):
        assert 0 < gq.ffn_gate_up_workspace_bytes(fmt, m, 64, k) <= 128 << 20
    for n in (16, 14336, 1 << 20, 1 << 22, 1 << 24):
        assert 0 < gq.ffn_gate_up_bwd_workspace_bytes(fmt, m, n, 256) <= 128 << 20


def test_binding_refuses_host_tensors_and_shapes():
    x = torch.zeros(2, 256)
    w = torch.zeros(1 << 16, dtype=torch.uint8)
    with pytest.raises(gq.GQError):
        gq.ffn_gate_up(gq.FMT_Q4_0, w, w, x, 64, 256)
    with pytest.raises(gq.GQError):
        gq.ffn_gate_up_bwd(gq.FMT_Q4_0, w, w, x, x, x, 256, 256)
    with pytest.raises(gq.GQError):
        gq.w4_gemv(w, 128, x, 64, 256)
    with pytest.raises(gq.GQError):
        gq.w4_gate_up(w, w, 128, x[0, :5], 64, 256)
    with pytest.raises(gq.GQError):
        gq.w4_pack(w.reshape(-1, 128)[:64], torch.zeros(64, 2, dtype=torch.float16), None, 64, 256, 128)


def act_grad(act, g):
    """act(g) and act'(g) as the header gives them, in 64 bits."""
    if act == gq.ACT_SILU:
        s = torch.sigmoid(g)
        return g * s, s * (1 + g * (1 - s))
    c = (2 / torch.pi) ** 0.5
    t = torch.tanh(c * (g + 0.044715 * g ** 3))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * c * (1 + 3 * 0.044715 * g * g)


@pytest.mark.parametrize("act", [gq.ACT_SILU, gq.ACT_GELU_TANH])
def test_gradient_formula_against_differences(act):
    gen = torch.Generator().manual_seed(act)
    x, wg, wu, dh = (torch.randn(*s, generator=gen, dtype=torch.float64) for s in ((3, 8), (5, 8), (5, 8), (3, 5)))

    def loss(x):
        return float(((act_grad(act, x @ wg.t())[0] * (x @ wu.t())) * dh).sum())

    f, d = act_grad(act, x @ wg.t())
    dx = (dh * (x @ wu.t()) * d) @ wg + (dh * f) @ wu
    for i in range(x.numel()):
        e = torch.zeros_like(x)
        e.view(-1)[i] = 1e-6
        assert abs((loss(x + e) - loss(x - e)) / 2e-6 - float(dx.view(-1)[i])) <= 1e-6 * (1 + abs(float(dx.view(-1)[i])))
