"""How far paged attention's output may be off as a whole, and its arithmetic in pieces on the host.

An element-wise bound has to allow every rounding its worst sign. Roundings of many tokens
do not conspire, so with random keys and values the norm of the error says far more:
o = sum w_j v_j / sum w_j, and relative errors d_j of the weights change it by
sum w_j (d_j - mean) v_j, whose norm is rms(d) times that of o.  Root mean squares, for
scores of standard deviation 1 and up to 4000 tokens, in units of 2^-24:
  exp2 of the approximate unit, 2 units of the result at most:                        4
  the score: up to D/32 + 8 truncations and roundings of sums of about 8 before the
    scale of D^-1/2, that is of 0.7 (D = 128) at most 2 units each, random in size:    3
  score times scale less maximum, up to 8 in units of log2, one rounding:             2
  pieces of p and q, 22 bits or more (both, and q's over a sum as large as the score): 3
  o and the sum of weights: half a unit a step, 4000 tokens in steps of 16 or 32,
    running sums below the last one: sqrt(250 / 2) / 2, and its joins:                 6
together sqrt(16 + 9 + 4 + 9 + 36) = 8.6 units = 5.1e-7.  NORM is twice that, 2^-20.
A lost third piece of q or p leaves 16 bits, off by up to 2^-17 of the leading bit: uniform
between mantissas, 2^-17 / sqrt(3) / 1.4 = 3.1e-6 rms, three times NORM.
"""
import math

import torch

NORM = 2.0 ** -20


def norm_error(got, want):
    return ((got.double() - want).norm() / want.norm()).item()


def cut(x, dtype, pieces):
    """The 16-bit pieces that the kernels make of f32 x, summed in 64 bits: the first `pieces` of them."""
    total, rest = torch.zeros_like(x, dtype=torch.float64), x.float()
    for _ in range(pieces):
        w = rest.to(dtype).float()
        total += w.double()
        rest = rest - w
    return total


def attention_in_pieces(q, k, v, scale, dtype, q_pieces, p_pieces):
    """[heads, D] of one row over its own [n, D] keys and values (16-bit values, all heads share them)."""
    up = torch.ones(q.shape[0], 1)
    if dtype is torch.float16:  # each head's largest element into [2^7, 2^8), as the kernel does
        up = torch.exp2(7 - torch.floor(torch.log2(q.abs().amax(-1, keepdim=True))))
    s = ((cut(q * up, dtype, q_pieces) / up.double()) @ k.double().T).float()
    s = (s * (scale * math.log2(math.e))).float()
    shift = 14.0 if dtype is torch.float16 else 0.0
    w = torch.exp2(s - s.amax(-1, keepdim=True) + shift)
    return cut(w, dtype, p_pieces) @ v.double() / w.double().sum(-1, keepdim=True)
