"""Bars on attention outputs that a lost, doubled or extra key breaks, for long caches.

A worst-case bound of every rounding (kv4_ref.attention's) exceeds the output itself there: with values of
mean zero an output over n keys shrinks as 1/sqrt(n).  Two other statements are used:

relative: the error's norm over a head's channels against the output's, values without a common mean.
    The output's own rounding is at most u in this norm (every element's is).  Before it, products take operands
    of 11 bits: a probability, and where a request has many rows the held key and value, each off by 0.43 * 2^-11
    = 2.1e-4 (rms) relatively, independently of one another.  Probabilities and values enter as they are; a key's
    error moves a score by scale * |q||k| rms, that is by k's rms value (1.6 for the tests' keys) times 2.1e-4.  Together
    4.5e-4; the bar takes 1e-3.  Leaving out m of n keys moves an output by about sqrt(m/n).

counts: a zero query gives every visible key the same probability, and key p's value is 15/16 in channel
    p // block of the head and 0 in the others, which the cache holds exactly; an output is then
    15/16 * (visible keys of the block) / (visible keys), whose products and sums are exact, so only the
    division and the output's rounding are off: (u + 2^-20) of it, where one key more or less is
    1/block of it.

beyond rounding: what an output is off by that its own rounding does not explain, over many outputs:
    sqrt(error^2 - rounding^2) of their norms against the outputs'.  A probability times step of 11 bits is off
    by 2.1e-4 (rms); where that counts against the value's own size it gives 2.1e-4 here.  64 normal channels span
    about 4.8 deviations, 15 steps: against the whole code (0 to 15) it would be 2.6 times as much, 5.5e-4.
    The bar is 3.2e-4, one and a half of the former.  F16 outputs, where operands are kept in two parts of 11
    bits, 2^-18 and less: what is left are f32 sums that the matrix unit cuts, each by 2^-24 of a sum that is
    tens to hundreds of times the output; the bar is 1e-4, half the output's own rounding, and below any one
    operand of 11 bits."""

import torch

UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def relative_bar(dtype):
    return UNIT[dtype] + 1e-3


def relative(got, want):
    """The error's norm over the last axis against want's, worst over the others."""
    return ((got.double() - want).norm(dim=-1) / want.norm(dim=-1)).max().item()


def count_values(n, d, device="cpu"):
    """Values [n, d] of the count statement, and the block's length."""
    block = -(-n // d)
    p = torch.arange(n, device=device)
    v = torch.zeros((n, d), device=device)
    v[p, p // block] = 15.0 / 16.0
    return v, block


def counts_at(pos, d, block, window=0):
    """The count statement's outputs [rows, d] (f64) of rows at positions `pos` (0 of a row before position 0)."""
    pos = pos[:, None].double()
    low = (pos - window + 1).clamp(min=0) if window else torch.zeros_like(pos)
    first = torch.arange(d, device=pos.device)[None, :].double() * block
    inside = (torch.minimum(pos + 1, first + block) - torch.maximum(low, first)).clamp(min=0)
    return 15.0 / 16.0 * inside / (pos - low + 1).clamp(min=1)


def counts(n, rows, d, block, window=0, device="cpu"):
    """Those of the last `rows` positions of n keys."""
    return counts_at(torch.arange(n - rows, n, device=device), d, block, window)


def count_bar(want, dtype):
    """The allowed error of each output (a channel without visible keys is 0 exactly): half the type's spacing, which
    for F16 does not shrink below 2^-24, and 2^-20 of it."""
    half = (want * UNIT[dtype]).clamp(min=2.0 ** -25 if dtype == torch.float16 else 0.0)
    return torch.where(want > 0, half + want * 2.0 ** -20, torch.zeros_like(want))


BEYOND_BAR = {torch.bfloat16: 3.2e-4, torch.float16: 1e-4}


def beyond_rounding(got, want):
    """sqrt(|error|^2 - |own rounding|^2) against |want|, over all outputs."""
    error = (got.double() - want).norm()
    own = (want.to(got.dtype).double() - want).norm()
    return (error.square() - own.square()).clamp(min=0).sqrt().item() / want.norm().item()
