"""CPU: the bound that expert layers in e4m3 are held to notices an intermediate that is not quantised as defined."""
import pytest
import torch

from fp8_layers import experts64, norm_bound, outliers
from fp8_reference import block_scales, e4m3, layer, rounded
from helpers import randn
from test_gpu_fp8_experts import routing


def truncated(h):
    """Codes cut off towards zero."""
    s = block_scales(h).repeat_interleave(128, dim=-1)
    v = h / s
    exponent = torch.frexp(v)[1] - 1
    step = torch.ldexp(torch.ones_like(v), exponent.clamp(min=-6) - 3)
    return torch.trunc(v / step) * step * s


def saturated(h):
    """A scale that is one power of two too small."""
    s = block_scales(h).repeat_interleave(128, dim=-1) / 2
    return e4m3((h / s).clamp(-448, 448)) * s


def neighbour(h):
    """The scale of the block beside it."""
    s = block_scales(h)
    codes = rounded(h) / s.repeat_interleave(128, dim=-1)
    return codes * s.roll(1, dims=-1).repeat_interleave(128, dim=-1)


WRONG = {"unquantised": lambda h: h, "truncated": truncated, "saturated": saturated, "twice the scale": lambda h: 2 * rounded(h), "another block's scale": neighbour}


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("factor", [1.0, 100.0])
@pytest.mark.parametrize("wrong", sorted(WRONG))
def test_the_bound_notices(wrong, factor, dtype):
    T, E, K, H, I = 40, 3, 2, 512, 1024
    _, _, w1, w2 = layer(E, H, I, T + 1)
    ids, wts = routing(T, E, K, dtype, T)
    x = outliers(randn((T, H), dtype, 1.0, T), factor).to(dtype)
    want = experts64(x, w1, w2, ids, wts)
    assert (want.to(dtype).double() - want).norm() <= norm_bound(dtype) * want.norm()
    got = experts64(x, w1, w2, ids, wts, WRONG[wrong]).to(dtype).double()
    assert (got - want).norm() > 2 * norm_bound(dtype) * want.norm()
