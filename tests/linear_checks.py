"""Checks of a gradient along directions in which it is large, for the tests of the product with its epilogue."""
import torch

DIFFERENCE = 2e-2  # the share of a derivative that a gradient may be off by (along_errors)
STEP = 2.0 ** -8   # of the size of what is moved


def directions(grad, ungated, like, seed=0):
    """Directions of the size of `like`: along the gradient and along the gradient without its activation's derivative, which differ
    where the derivative does, each with a fixed random part."""
    gen = torch.Generator().manual_seed(seed)
    size = float(like.double().norm())
    out = []
    for g in (grad, ungated):
        r = torch.randn(g.shape, generator=gen, dtype=torch.float64).to(g.device)
        v = g.double() / g.double().norm() + 0.3 * r / r.norm()
        out.append(v * (size / v.norm()))
    return out


def off_the_kink(act, z, dy):
    """dy, for ReLU zero where z is so near 0 that a step could cross it (differences across it are of neither slope)."""
    return torch.where(z.abs() < 0.5, 0.0, dy) if act == 3 else dy


def along_errors(loss, at, grad, along, e=STEP):
    """For each direction v: how far the gradient's product with v is from the central difference of loss around `at`, as a share of
    that difference.  loss takes what `at` is moved to, in 64 bits."""
    errors = []
    for v in along:
        d = (loss(at.double() + e * v) - loss(at.double() - e * v)) / (2 * e)
        errors.append(abs(float((grad.double() * v).sum()) - d) / abs(d))
    return errors


def wrong(grad, ungated):
    """Gradients that a check has to refuse: negated, halved, without the activation's derivative, of half the rows, noise of the same size."""
    gen = torch.Generator().manual_seed(1)
    noise = torch.randn(grad.shape, generator=gen, dtype=torch.float64).to(grad.device)
    half = grad.double().clone()
    half[: (len(half) + 1) // 2] = 0
    return {"negated": -grad.double(), "halved": grad.double() / 2, "ungated": ungated.double(), "half": half,
            "noise": noise * (grad.double().norm() / noise.norm())}
