"""The formulas of the product with its epilogue in 64 bits, for the tests."""
import math

import torch

import gq


def act_grad(act, z):
    """act(z) and act'(z) of a float64 tensor."""
    if act == gq.ACT_NONE:
        return z, torch.ones_like(z)
    if act == gq.ACT_RELU:
        return z.clamp(min=0), (z > 0).double()
    if act == gq.ACT_SILU:
        s = torch.sigmoid(z)
        return z * s, s + z * s * torch.sigmoid(-z)
    p = 2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)
    s = torch.sigmoid(p)
    return z * s, s + z * s * torch.sigmoid(-p) * 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * z ** 2)
