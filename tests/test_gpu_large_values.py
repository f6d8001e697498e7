"""The largest values of x that the header allows where x enters the matrix cores unscaled, in the sums that are largest there:
every value of one sign next to the bound, every code the largest, so that the sums of codes with their
offset come closest to fp32's limit.

Tolerances: 2^-7 of the value.  x is equal along a row, so sums of x are exact but for fp32 roundings (2^-24 each, at
most 47 / 7 times the result's size and a few hundred of them: 2e-4), the weights are exact powers of two, and the
output is fp32."""
import os
import re

import numpy as np
import pytest
import torch

import oracle as O

pytestmark = pytest.mark.gpu
HEADER = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include", "gq.h")


def bounds():
    """The exponents N of the header's "finite values must stay below 2^N", the front's and the 4-bit products'."""
    text = re.sub(r"\s+\*?\s*", " ", open(HEADER).read())
    found = [int(e) for e in re.findall(r"finite values must stay below 2\^(\d+)", text)]
    assert len(found) == 2
    return found


def below(exponent):
    """The largest bf16 below 2^exponent."""
    return 2.0 ** exponent * (1 - 2.0 ** -8)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [1, 4, 5, 16])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("zero", [0, 31])
def test_w4(dev, dtype, m, group, zero):
    import gq
    n, k = 20, 256
    x = torch.full((m, k), below(bounds()[1]), dtype=dtype, device=dev)
    assert bool(x.isfinite().all())
    q = torch.full((n, k // 2), 0xFF, dtype=torch.uint8, device=dev)
    s = torch.full((n, k // group), 2.0 ** -14, dtype=torch.float16, device=dev)
    z = torch.full((n, k // group), zero, dtype=torch.uint8, device=dev)
    y = gq.w4_gemv(gq.w4_pack(q, s, z, n, k, group), group, x, n, k, out_dtype=torch.float32)
    want = k * float(x[0, 0]) * (15 - zero) * 2.0 ** -14
    assert float((y.double() / want - 1).abs().max()) <= 2.0 ** -7


@pytest.mark.parametrize("fmt", [O.Q4_0, O.Q8_0, O.Q4_K, O.Q6_K])
@pytest.mark.parametrize("m", [1, 4, 5, 16, 40])
@pytest.mark.parametrize("k", [512, 4608])
def test_front(dev, fmt, m, k):
    import gq
    n = 20
    x = torch.full((m, k), below(bounds()[0]), dtype=torch.bfloat16, device=dev)
    blocks = O.gen_weights(fmt, n, k, seed=1).reshape(-1, {O.Q4_0: 18, O.Q8_0: 34, O.Q4_K: 144, O.Q6_K: 210}[fmt])
    # every code its largest value; scales a power of two, no minima
    half = np.frombuffer(np.float16(2.0 ** -14).tobytes(), np.uint8)
    if fmt in (O.Q4_0, O.Q8_0):
        blocks[:, :2], blocks[:, 2:] = half, 0xFF if fmt == O.Q4_0 else 0x7F
    elif fmt == O.Q4_K:
        blocks[:, 0:2], blocks[:, 2:4], blocks[:, 16:] = half, 0, 0xFF
        blocks[:, 4:16] = np.uint8(1)
    else:
        blocks[:, :192], blocks[:, 192:208], blocks[:, 208:] = 0xFF, 1, half
    w = O.dequant(fmt, np.ascontiguousarray(blocks).reshape(-1)).reshape(n, k)
    assert np.isfinite(w).all() and (w >= 0).all() and (w.max(axis=1) > 0).all()
    p = gq.repack(fmt, torch.from_numpy(np.ascontiguousarray(blocks).reshape(-1)).to(dev), n, k)
    _, g, u = gq.ffn_gate_up(fmt, p, p, x, n, k, save=True, out_dtype=torch.float32)
    want = x.double() @ torch.from_numpy(w).to(dev).double().t().contiguous()
    assert float((g.double() / want - 1).abs().max()) <= 2.0 ** -7 and torch.equal(g, u)
