"""bf16 rows of the product with its epilogue and of the experts next to the bound of those that enter the matrix cores unscaled, 2^115: every
value of one sign, every code the largest (as test_gpu_large_values for the front).  Tolerance as there: 2^-7 of the value."""
import numpy as np
import pytest
import torch

import oracle as O
from test_gpu_large_values import below

pytestmark = pytest.mark.gpu
FMTS = [O.Q4_0, O.Q8_0, O.Q4_K, O.Q6_K]


def largest(fmt, n, k, scale=2.0 ** -14):
    """Blocks whose codes are all the largest; scales a power of two, no minima."""
    blocks = O.gen_weights(fmt, n, k, seed=1).reshape(-1, {O.Q4_0: 18, O.Q8_0: 34, O.Q4_K: 144, O.Q6_K: 210}[fmt])
    half = np.frombuffer(np.float16(scale).tobytes(), np.uint8)
    if fmt in (O.Q4_0, O.Q8_0):
        blocks[:, :2], blocks[:, 2:] = half, 0xFF if fmt == O.Q4_0 else 0x7F
    elif fmt == O.Q4_K:
        blocks[:, 0:2], blocks[:, 2:4], blocks[:, 4:16], blocks[:, 16:] = half, 0, 1, 0xFF
    else:
        blocks[:, :192], blocks[:, 192:208], blocks[:, 208:] = 0xFF, 1, half
    b = np.ascontiguousarray(blocks).reshape(-1)
    return b, O.dequant(fmt, b).reshape(n, k)


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", [1, 3, 4, 5, 16, 40])
@pytest.mark.parametrize("k", [512, 4608])
def test_product(dev, fmt, m, k):
    import gq
    n = 20
    b, w = largest(fmt, n, k)
    assert np.isfinite(w).all() and (w >= 0).all() and (w.max(axis=1) > 0).all()
    x = torch.full((m, k), below(115), dtype=torch.bfloat16, device=dev)
    y = gq.linear(fmt, gq.repack(fmt, torch.from_numpy(b).to(dev), n, k), x, n, k, out_dtype=torch.float32)
    want = x.double() @ torch.from_numpy(w).to(dev).double().t().contiguous()
    assert float((y.double() / want - 1).abs().max()) <= 2.0 ** -7


@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("m", [1, 4, 5, 40])
def test_experts(dev, fmt, m):
    """x at the bound in one column where the gate's weights are ordinary and u's are zeros: h = 0 is right, an Inf would make it a NaN; and
    at 2^58, with all codes the largest, h = g u of 2^116 and more."""
    import gq
    e, n, k = 2, 256, 512
    b, w = largest(fmt, e * n, k)
    zero = gq.repack(fmt, torch.zeros(gq.gguf_bytes(fmt, e * n, k), dtype=torch.uint8, device=dev), e * n, k)
    p = gq.repack(fmt, torch.from_numpy(b).to(dev), e * n, k)
    db, dw = largest(O.Q8_0, e * k, n, 2.0 ** -24)
    down = gq.repack(O.Q8_0, torch.from_numpy(db).to(dev), e * k, n)
    ids, weights = torch.zeros(m, 1, dtype=torch.int32, device=dev), torch.ones(m, 1, device=dev)
    x = torch.full((m, k), below(115), dtype=torch.bfloat16, device=dev)
    y = gq.moe_ffn(fmt, p, zero, O.Q8_0, down, x, ids, weights, n, k, e, out_dtype=torch.float32)
    assert bool((y == 0).all())
    x = torch.full((m, k), 2.0 ** 58, dtype=torch.bfloat16, device=dev)
    y = gq.moe_ffn(fmt, p, p, O.Q8_0, down, x, ids, weights, n, k, e, out_dtype=torch.float32)
    g = x.double() @ torch.from_numpy(w[:n]).to(dev).double().t().contiguous()
    want = (g * g) @ torch.from_numpy(dw[:k]).to(dev).double().t().contiguous()
    assert 2.0 ** 90 < float(want.max()) < 2.0 ** 127 and float((y.double() / want - 1).abs().max()) <= 2.0 ** -7
