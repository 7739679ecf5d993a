"""Whole expert layers in e4m3 from their definition in 64 bits, an expert at a time, and how far a layer's result may be from it in the 2-norm."""
import math

import torch

from fp8_reference import HALF, rounded


def outliers(x, factor):
    """One column of each block of 128 far larger than the others, as activations of a language model have them."""
    x = x.float()
    x[:, 5::128] *= factor
    return x


def experts64(x, w1, w2, ids, wts, quantise=rounded):
    """y [T, H] in 64 bits.  `quantise`: what the intermediate goes through."""
    xq, inter = rounded(x), w2.shape[2]
    y = torch.zeros(x.shape, dtype=torch.float64)
    for e in range(w1.shape[0]):
        token, pick = (ids == e).nonzero(as_tuple=True)
        if token.numel() == 0:
            continue
        both = xq[token] @ w1[e].t()
        h = quantise(torch.nn.functional.silu(both[:, :inter]) * both[:, inter:])
        y.index_add_(0, token, (h @ w2[e].t()) * wts[token, pick].double().unsqueeze(1))
    return y


def norm_bound(dtype):
    """How far a result may be off, of its own 2-norm.  Rounding: a step is 2 HALF of a number at most and the error is even over it, step / sqrt(12).  Codes that move: gate and up of 512 k are some 20 roundings
    of fp32 each, sqrt(20) 2^-24 / sqrt(3) of a sum, together eps = 4 2^-24 of an intermediate; that is across a border of codes with probability 2 eps |h| / step and costs a step, which is
    0.09 |h| in the mean of its logarithm, so sqrt(2 0.09 eps) of the norm.  Both are sums over many independent errors."""
    return math.sqrt((2 * HALF[dtype]) ** 2 / 12 + 2 * 0.09 * 4 * 2.0 ** -24)
