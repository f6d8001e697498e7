"""Every kernel that the gated front's plan can take, in every format and type of x, at shapes that end inside its tiles.

Beside each shape stands the kernel it is for (row tiles are of 16 rows of the weights, units of 128 k).  Tolerances are
those of test_gpu_ffn; one to four rows of 16 bits have fp32 sums alone: the codes carry an offset of up to 1152, 224 times
their spread of 4.6 in the worst format, and a scale group's sum takes up to four roundings of 2^-24 of that size:
4 * 224 * 2^-24 = 5e-5 of its norm, 1e-4 with the sums over groups."""
import pytest
import torch

import oracle as O
from test_gpu_ffn import DTYPES, Case, check_front, check_grads, half_step, worst_row

pytestmark = pytest.mark.gpu
FMTS = [O.Q4_0, O.Q8_0, O.Q4_K, O.Q6_K]
SUMS = 1e-4

SHAPES = [
    # k_front_few_px: 1..4 rows of 16 bits, up to 32 units (fp32: k_front_rows_px); 8, 16, 32 units; more row tiles than CUs
    (1, 200, 768), (3, 170, 768), (4, 83, 1280), (1, 90, 2048), (2, 4200, 2048), (1, 4113, 2304), (3, 130, 4096),
    # k_front_few: more units; up to 256 row tiles, up to 448, more (fp32 and odd addresses: a conversion first)
    (1, 300, 4352), (3, 301, 4608), (1, 5000, 4352), (4, 4999, 4352), (1, 7300, 4352), (2, 7201, 4608),
    # k_front_rows_px: 5..16 rows up to 32 units, 17..32 up to 16; 8, 16, 32 units; more row tiles than CUs
    (9, 100, 1024), (5, 200, 1280), (16, 4200, 2048), (11, 4200, 4096), (16, 77, 2304), (20, 4200, 2048), (31, 200, 1280),
    (32, 90, 768),
    # k_front_rows: 5..16 rows of more units, up to 448 row tiles and more; 17..32 rows, up to 400 row tiles
    (11, 4200, 4352), (16, 7300, 4352), (24, 1000, 2304), (32, 6399, 2304),
    # k_front_rb<32, 2, 1, 4, 4>: 17..32 rows, more row tiles
    (30, 6500, 2304), (17, 6401, 4096),
    # <64, 2, 1, 3, 4>, <64, 4, 1, 3, 2>, <128, 4, 1, 3, 2>, <128, 4, 1, 2, 1>
    (61, 1000, 1024), (130, 9001, 512), (250, 12000, 512), (2043, 4100, 512),
]
# K that is no whole chunk of the layout, and (the last two) an odd number of pairs of steps: no four K groups
SHORT = [(1, 300, 4128), (3, 7300, 4128), (11, 300, 4192), (24, 100, 2208), (30, 6500, 2176), (60, 500, 160)]


def run(dev, fmt, m, n, k):
    import gq
    c = Case(dev, fmt, m, n, k, seed=n)
    x = c.x
    for i, dtype in enumerate(DTYPES):
        c.x = x.to(dtype)
        act = (m + i) % 2
        out = gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, act=act, save=True)
        check_front(c, act, out, dtype)
        # the same at an odd address, and with fp32 outputs
        odd = torch.empty(m * k + 1, dtype=dtype, device=dev)[1:].view(m, k).copy_(c.x)
        full = gq.ffn_gate_up(fmt, *c.packed, odd, n, k, act=act, save=True, out_dtype=torch.float32)
        check_front(c, act, full, torch.float32)
        if m <= 4 and dtype != torch.float32:
            _, g, u = gq.ffn_gate_up(fmt, *c.packed, c.x, n, k, act=act, save=True, out_dtype=torch.float32)
            _, rg, ru = c.front(act)
            assert worst_row(g, rg) <= SUMS + half_step(torch.float32) and worst_row(u, ru) <= SUMS + half_step(torch.float32)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_front_kernels(dev, fmt, m, n, k):
    run(dev, fmt, m, n, k)


@pytest.mark.parametrize("fmt", [O.Q4_0, O.Q8_0])
@pytest.mark.parametrize("m,n,k", SHORT)
def test_front_short_chunks(dev, fmt, m, n, k):
    run(dev, fmt, m, n, k)


# k_front_dx<1, 4, 1>, <1, 4, 2>, <2, 2, 4> with the sum over the weights' rows in one part and in several
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1000, 256), (32, 500, 14336 * 2), (29, 4099, 512), (33, 200, 16384), (128, 3001, 768),
                                   (129, 70, 512), (300, 2050, 1024), (1000, 130, 8192)])
def test_backward_kernels(dev, fmt, dtype, m, n, k):
    import gq
    c = Case(dev, fmt, m, n, k, seed=n, dtype=dtype)
    check_grads(c, 1, gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k, act=1), dtype)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n", [16383, 16384, 16385, 33001])
def test_backward_of_long_rows_in_place(dev, dtype, n):
    """Columns past those that stay in registers are computed twice, here with dg over g and du over u."""
    import gq
    fmt, m, k = O.Q8_0, 5, 64
    c = Case(dev, fmt, m, n, k, seed=n, dtype=dtype)
    full = gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, c.g, c.u, n, k)
    check_grads(c, 0, full, dtype)
    g, u = c.g.clone(), c.u.clone()
    out = gq.ffn_gate_up_bwd(fmt, *c.packed, c.dh, g, u, n, k, dg=g, du=u)
    assert torch.equal(g, full["dg"]) and torch.equal(u, full["du"]) and torch.equal(out["dx"], full["dx"])
