"""What the products' roundings come to, path by path, as a share of the root of a row's sum of squared terms, for the tests.

A rounding to fp16 is uniform within a half step: 2^-11 / sqrt(3) of a term of mantissa 1, 0.72 of that in the mean square
over mantissas, 2.03e-4.  Independent roundings add by squares.  SPREAD: a norm over 100 columns and more is within a quarter of the mean.
fp32 sums: a group of 32 terms x (OFF + q) adds 32 partial sums that grow as a root, each rounded or cut by up to a step of 2^-24 to 2^-23,
and the same again for OFF sum x: 1.95e-7 (OFF / size of q + 1) of the group's terms; twice that, with the sums of the groups' sums."""
import torch

import oracle as O

HALF = 2.03e-4
SPREAD = 1.25
CODES = {O.Q4_0: 4.6, O.Q8_0: 73.3, O.Q4_K: 4.6, O.Q6_K: 18.5}  # root mean square of uniform codes around their middle


def padded(fmt, k):
    unit = 128 if fmt in (O.Q4_0, O.Q8_0) else 256
    return -(-k // unit) * unit


def few(fmt, dtype):
    """One to four rows: fp32 sums."""
    bf16 = dtype == torch.bfloat16
    off = {O.Q4_0: 8, O.Q8_0: 0 if bf16 else 128, O.Q4_K: 0, O.Q6_K: 32}[fmt] + (0 if bf16 and fmt == O.Q8_0 else 128 if bf16 else 1024)
    return 2 * 1.95e-7 * (off / CODES[fmt] + 1)


def rows(fmt):
    """Up to 16 rows, and the experts' products of more than four tokens: weights of Q4_0 and Q8_0 once to fp16; the k-quants' codes
    times their scales' codes are exact (of these tests' Q6_K scales, up to 32), their d and minima are fp32; a unit of 128 terms."""
    return SPREAD * HALF * (fmt in (O.Q4_0, O.Q8_0)) + 4e-6


def tiles(fmt):
    """More rows: k-quants fold d too.  Q6_K rounds twice, Q4_K its minimum, up to three times the weight, and the weight."""
    return SPREAD * HALF * {O.Q4_0: 1, O.Q8_0: 1, O.Q6_K: 2, O.Q4_K: 10}[fmt] ** 0.5 + 4e-6


def taken(x):
    """What the matrix cores take of fp32 rows: fp16 after a power of two per row.  (Of 16-bit rows they take the values themselves.)  Held apart
    from the shares, since its errors are the same in all columns: where these have a common part, the norm over the columns of their sum is one
    normal variable, not the mean of many."""
    if x.dtype != torch.float32:
        return x.double()
    s = torch.exp2(14 - x.double().abs().amax(1, keepdim=True).clamp(min=2.0 ** -126).log2().floor())
    return (x.double() * s).float().half().double() / s


def linear(fmt, m, k, dtype):
    if m <= 4 and m * padded(fmt, k) <= 65536:
        return few(fmt, dtype)
    return rows(fmt) if m <= 16 else tiles(fmt)


def terms(x, w):
    """The root of the sum of squared terms of x W^T, per row, in the mean square over the columns, times the root of their number."""
    return (x.double().pow(2) @ w.double().pow(2).t().contiguous()).sum(1).sqrt()
