"""The shares of figures by themselves: weights rounded to fp16 once, twice or not at all, in 64 bits, against the bound of each path.  A kernel
of few rows that rounded its weights would miss its bound, whatever its sums do."""
import pytest
import torch

import figures
import oracle as O


@pytest.mark.parametrize("fmt", [O.Q4_0, O.Q8_0, O.Q4_K, O.Q6_K])
@pytest.mark.parametrize("k", [512, 4096])
def test_rounded_weights(fmt, k):
    n, m = 160, 4
    w = torch.from_numpy(O.dequant(fmt, O.gen_weights(fmt, n, k, seed=k)).reshape(n, k)).double()
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(m, k, generator=gen, dtype=torch.float64).half().double()
    share = float(((x @ (w.half().double() - w).t()).norm(dim=1) / figures.terms(x, w)).min())
    most = float(((x @ (w.half().double() - w).t()).norm(dim=1) / figures.terms(x, w)).max())
    for dtype in (torch.float16, torch.bfloat16):
        assert share > 1.5 * figures.few(fmt, dtype)
    assert most <= figures.tiles(fmt)
    if fmt in (O.Q4_0, O.Q8_0):
        assert most <= figures.rows(fmt)
    else:
        assert share > 10 * figures.rows(fmt)


def test_what_is_taken_of_fp32_rows():
    x = torch.randn(5, 64) * torch.tensor([1.0, 2.0 ** 100, 2.0 ** -100, 0.0, 1e-30])[:, None]
    t = figures.taken(x)
    assert bool(((t - x.double()).abs() <= 2.0 ** -11 * x.double().abs()).all())
    assert torch.equal(figures.taken(x.half()), x.half().double())
