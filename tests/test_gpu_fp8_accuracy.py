"""GPU: results of the e4m3 expert layers are as good as their rounding, whichever plan a call takes, and with outlying columns too."""
import pytest
import torch

from fp8_layers import experts64, norm_bound, outliers
from fp8_reference import layer
from helpers import randn
from test_gpu_fp8_experts import on_gpu, routing

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("factor", [1.0, 30.0, 100.0])
@pytest.mark.parametrize("T", [1, 9, 40, 130, 300, 700])
def test_layers_are_as_good_as_their_rounding(mlk, T, factor, dtype):
    """One token, streamed, and panels of every width.  With gate and up from sums of 13 bits, as the 8-bit products leave them, bf16 layers of 130 tokens and more with such columns are
    2.3e-3 to 3.4e-3 off, where 2.26e-3 are allowed."""
    E, K, H, I = 3, 2, 512, 1024
    l1, l2, w1, w2 = layer(E, H, I, T + 1)
    a1, a2, s1, s2 = on_gpu(mlk, l1, l2)
    ids, wts = routing(T, E, K, dtype, T)
    x = outliers(randn((T, H), dtype, 1.0, T), factor).to(dtype)
    got = mlk.fused_experts_fp8(x.cuda(), a1, a2, ids.cuda(), wts.cuda(), s1, s2).cpu().double()
    want = experts64(x, w1, w2, ids, wts)
    assert (got - want).norm() <= norm_bound(dtype) * want.norm()


@pytest.mark.parametrize("factor", [1.0, 100.0])
def test_a_layer_through_the_queues(mlk, factor):
    """8 experts with very different loads, an intermediate long enough for two slices of the down projection."""
    T, E, K, H, I = 300, 8, 2, 1024, 8192
    g = torch.Generator().manual_seed(7)
    l1, l2, w1, w2 = layer(E, H, I, 11)
    a1, a2, s1, s2 = on_gpu(mlk, l1, l2)
    ids = (torch.rand((T, E), generator=g) + torch.rand(E, generator=g) * 0.6).topk(K, dim=-1)[1].int()
    wts = (torch.rand((T, K), generator=g) + 0.1).to(BF)
    x = outliers(randn((T, H), BF, 1.0, 3), factor).to(BF)
    got = mlk.fused_experts_fp8(x.cuda(), a1, a2, ids.cuda(), wts.cuda(), s1, s2).cpu().double()
    want = experts64(x, w1, w2, ids, wts)
    assert (got - want).norm() <= norm_bound(BF) * want.norm()
