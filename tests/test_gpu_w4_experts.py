"""GPU: expert layers over 4-bit weights (`fused_experts_w4`, `fused_moe_w4`) against 64 bits on the CPU."""
import pytest
import torch

from helpers import randn
from test_gpu_w4 import centred_weights, on_gpu, w4_weights

pytestmark = pytest.mark.gpu


def layer(E, H, I, group, dtype, zeros, seed):
    c1, s1, z1, w1 = w4_weights(2 * I, H, group, dtype, zeros, seed, (E,))
    c2, s2, z2, w2 = w4_weights(H, I, group, dtype, zeros, seed + 1, (E,))
    return (c1, s1, z1), (c2, s2, z2), w1, w2


def routing(T, E, K, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    logits = torch.randn((T, E), generator=g) + torch.randn(E, generator=g)
    p, ids = torch.topk(torch.softmax(logits, dim=-1), K)
    return ids.to(torch.int32).contiguous(), (p / p.sum(dim=-1, keepdim=True)).to(dtype)


def expected(x, w1, w2, s1, s2, ids, wts, emap=None):
    """y in 64 bits and how far a result may be off: the intermediate is rounded once (half a step), each product's fp32 sums by k / 64 2^-24 of
    62 sum |s x| (see the product's tests), and |d silu(g) / dg| < 1.1; the output is rounded once.  And the variance of the error: a rounding to
    nearest is off by at most half a step, evenly spread, so its variance is at most (half |value|)^2 / 3; the roundings of the intermediate's elements
    are independent and reach output n through W2[n, i] and the token's weight for the expert (the sum of them where it is picked twice)."""
    T, H = x.shape
    I = w2.shape[2]
    dtype = x.dtype
    half = torch.finfo(dtype).eps / 2
    y, tol, var = (torch.zeros(T, H, dtype=torch.float64) for _ in range(3))
    local = ids.long() if emap is None else torch.where((ids >= 0) & (ids < emap.numel()), emap[ids.long().clamp(0, emap.numel() - 1)].long(), -1)
    for e in range(w1.shape[0]):
        t, k = (local == e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        xe = x[t].double()
        both = xe @ w1[e].t()
        d = 62 * (xe.abs() @ s1[e].double().abs().repeat_interleave(H // s1.shape[2], dim=1).t()) * (H / 64) * 2.0 ** -24
        g, u = both[:, :I], both[:, I:]
        silu = g * torch.sigmoid(g)
        h = silu * u
        dh = 1.1 * d[:, :I] * u.abs() + silu.abs() * d[:, I:] + half * h.abs() + (2.0 ** -25 if dtype == torch.float16 else 0)
        wt = wts[t, k].double().unsqueeze(1)
        y.index_add_(0, t, wt * (h @ w2[e].t()))
        size2 = 62 * (h.abs() @ s2[e].double().abs().repeat_interleave(I // s2.shape[2], dim=1).t()) * (I / 64) * 2.0 ** -24
        tol.index_add_(0, t, wt * (dh @ w2[e].abs().t() + size2))
        share = torch.zeros(T, 1, dtype=torch.float64).index_add_(0, t, wt)
        hh = torch.zeros(T, I, dtype=torch.float64)
        hh[t] = h
        var += share ** 2 * ((half * hh) ** 2 / 3 @ (w2[e] ** 2).t())
    return y, tol + half * (y.abs() + tol) + 2.0 ** -25, var + (half * y) ** 2 / 3


def check(got, expect, dtype, what):
    want, tol, var = expect
    d = (got.cpu().double() - want).abs()
    assert (d <= tol).all(), "%s: off by %g more than allowed" % (what, (d - tol).max().item())
    # the errors' 2-norm is that of their variances, give or take chance (an output's errors share the intermediate's): half as much again
    if want.numel() > 1000:
        assert d.norm() <= 1.5 * var.sum().sqrt() + 1e-6 * want.norm(), "%s: 2-norm %g, %g expected" % (what, d.norm(), var.sum().sqrt())


@pytest.mark.parametrize("T", [1, 2, 3, 17, 40, 90, 200, 700])
@pytest.mark.parametrize("E,K,H,I,group,zeros,dtype", [
    (8, 2, 256, 384, 128, False, torch.bfloat16), (5, 3, 384, 256, 32, True, torch.float16), (40, 8, 128, 128, 64, True, torch.bfloat16),
    (1, 1, 512, 256, 256, False, torch.float16), (16, 4, 640, 1152, 128, True, torch.bfloat16)])
def test_experts_against_64_bits(mlk, T, E, K, H, I, group, zeros, dtype):
    p1, p2, w1, w2 = layer(E, H, I, group, dtype, zeros, 10 * E + T)
    x = randn((T, H), dtype, 1.0, T)
    ids, wts = routing(T, E, K, dtype, T + 7)
    (a1, s1, z1), (a2, s2, z2) = mlk.pack_layout_a_w4(*on_gpu(*p1)), mlk.pack_layout_a_w4(*on_gpu(*p2))
    got = mlk.fused_experts_w4(x.cuda(), a1, a2, ids.cuda(), wts.cuda(), s1, s2, z1, z2)
    want = expected(x, w1, w2, p1[1], p2[1], ids, wts)
    check(got, want, dtype, "experts")


@pytest.mark.parametrize("T", [1, 4, 60, 300])
def test_dropped_pairs_and_tokens_without_experts(mlk, T):
    E, held, K, H, I, dtype = 12, 5, 3, 256, 128, torch.bfloat16
    p1, p2, w1, w2 = layer(held, H, I, 64, dtype, True, T)
    x = randn((T, H), dtype, 1.0, T)
    ids, wts = routing(T, E, K, dtype, T)
    emap = torch.full((E,), -1, dtype=torch.int32)
    emap[torch.tensor([1, 4, 6, 9, 11])] = torch.tensor([3, 0, 4, 1, 2], dtype=torch.int32)
    ids[0] = torch.tensor([0, 2, 3], dtype=torch.int32)                 # all of them elsewhere
    if T > 3:
        ids[1] = torch.tensor([-1, E, 1 << 30], dtype=torch.int32)      # nobody's
        ids[2] = torch.tensor([4, 4, -5], dtype=torch.int32)            # the same one twice
    (a1, s1, z1), (a2, s2, z2) = mlk.pack_layout_a_w4(*on_gpu(*p1)), mlk.pack_layout_a_w4(*on_gpu(*p2))
    got = mlk.fused_experts_w4(x.cuda(), a1, a2, ids.cuda(), wts.cuda(), s1, s2, z1, z2, experts_map=emap.cuda())
    want = expected(x, w1, w2, p1[1], p2[1], ids, wts, emap)
    assert torch.equal(got[0].cpu(), torch.zeros(H, dtype=dtype))
    check(got, want, dtype, "experts here")
    if T > 3:
        assert torch.equal(got[1].cpu(), torch.zeros(H, dtype=dtype))


def test_a_token_with_nan_or_infinity_keeps_to_itself(mlk):
    E, K, H, I, dtype = 6, 2, 256, 256, torch.bfloat16
    p1, p2, w1, w2 = layer(E, H, I, 128, dtype, False, 1)
    (a1, s1, z1), (a2, s2, z2) = mlk.pack_layout_a_w4(*on_gpu(*p1)), mlk.pack_layout_a_w4(*on_gpu(*p2))
    for T in (5, 70, 400):
        x = randn((T, H), dtype, 1.0, T)
        ids, wts = routing(T, E, K, dtype, T)
        clean = mlk.fused_experts_w4(x.cuda(), a1, a2, ids.cuda(), wts.cuda(), s1, s2)
        x[1, 3], x[T - 1, 0] = float("nan"), float("inf")
        got = mlk.fused_experts_w4(x.cuda(), a1, a2, ids.cuda(), wts.cuda(), s1, s2)
        rest = torch.ones(T, dtype=torch.bool)
        rest[1] = rest[T - 1] = False
        assert torch.equal(got[rest.cuda()], clean[rest.cuda()])
        assert got[1].isnan().all()


def test_layer_router_counts_and_experts_together(mlk):
    from muxi_layout_kernels.muxi_moe_planC import fused_moe_w4
    E, K, H, I, dtype = 16, 4, 256, 256, torch.bfloat16
    p1, p2, w1, w2 = layer(E, H, I, 128, dtype, True, 3)
    (a1, s1, z1), (a2, s2, z2) = mlk.pack_layout_a_w4(*on_gpu(*p1)), mlk.pack_layout_a_w4(*on_gpu(*p2))
    load, total = torch.zeros(E, dtype=torch.int32, device="cuda"), torch.zeros(E, dtype=torch.int64)
    for T in (1, 9, 130):
        x, logits, bias = randn((T, H), dtype, 1.0, T), randn((T, E), dtype, 1.0, T + 1), randn((E,), dtype, 0.1, T + 2)
        y = fused_moe_w4(x.cuda(), a1, a2, logits.cuda(), K, True, s1, s2, z1, z2, True, 4, 2, bias.cuda(), "sigmoid", expert_load=load)
        ids = torch.empty((T, K), dtype=torch.int32, device="cuda")
        wts = torch.empty((T, K), dtype=dtype, device="cuda")
        mlk.fused_routing_gate(logits.cuda(), 1, T, H, 4, 2, ids, wts, K, bias.cuda(), True)
        assert torch.equal(y, mlk.fused_experts_w4(x.cuda(), a1, a2, ids, wts, s1, s2, z1, z2))
        want = expected(x, w1, w2, p1[1], p2[1], ids.cpu(), wts.cpu())
        check(y, want, dtype, "layer")
        total += torch.bincount(ids.cpu().flatten().long(), minlength=E)
        loss, counts = mlk.moe_balance_loss(logits.cuda(), ids, "sigmoid")
        assert torch.equal(counts.cpu().long(), torch.bincount(ids.cpu().flatten().long(), minlength=E))
        assert torch.isfinite(loss)
    assert torch.equal(load.cpu().long(), total)


@pytest.mark.parametrize("T", [1, 5, 40, 400])
def test_an_intermediate_past_the_range_of_fp16_is_nan_in_its_row(mlk, T):
    """A gate and an up of some hundred each: their product has no place in fp16.  One token, few, tasks of two blocks, panels."""
    E, K, H, I, dtype = 6, 2, 256, 256, torch.float16
    p1, p2, w1, _ = layer(E, H, I, 128, dtype, True, 1)
    (a1, s1, z1), (a2, s2, z2) = mlk.pack_layout_a_w4(*on_gpu(*p1)), mlk.pack_layout_a_w4(*on_gpu(*p2))
    x, (ids, wts) = randn((T, H), dtype, 1.0, T), routing(T, E, K, dtype, T)
    call = lambda: mlk.fused_experts_w4(x.cuda(), a1, a2, ids.cuda(), wts.cuda(), s1, s2, z1, z2)
    clean = call()
    assert torch.isfinite(clean).all()
    t = T // 2
    x[t] *= 2000.0
    g, u = (w1[ids[t, 0].long()] @ x[t].double()).split(I)
    assert torch.isfinite(x).all() and (g * torch.sigmoid(g) * u).abs().max() > 2 * 65504
    got = call()
    assert got[t].isnan().all() and torch.equal(got[:t], clean[:t]) and torch.equal(got[t + 1:], clean[t + 1:])


@pytest.mark.parametrize("mean", [0.0, 1.0, 20.0])
@pytest.mark.parametrize("T,group,zeros", [(300, 128, False), (90, 32, True), (5, 32, True)])
def test_error_does_not_grow_with_the_mean_of_the_activations(mlk, T, group, zeros, mean):
    """One expert in fp16, panels of 128 and of 64 tokens and few tokens: the error's 2-norm is that of the two roundings, of the intermediate and of the result, give or take a
    twentieth.  The fp32 sums are off by 2.2e-5 of gate and up (as derived at the products), some 5e-5 of the intermediate, beside the roundings' sqrt(2) * 2e-4: sqrt(1 + 0.03) = 1.02."""
    H, I = 14336, 128
    parts = [centred_weights(2 * I, H, group, zeros, 1), centred_weights(H, I, group, zeros, 2)]
    (a1, s1, z1), (a2, s2, z2) = [mlk.pack_layout_a_w4(*[None if t is None else t.unsqueeze(0).cuda() for t in p[:3]]) for p in parts]
    x = (randn((T, H), torch.float32, 1.0, 3) + mean).half()
    ids, wts = torch.zeros((T, 1), dtype=torch.int32, device="cuda"), torch.ones((T, 1), dtype=torch.float16, device="cuda")
    got = mlk.fused_experts_w4(x.cuda(), a1, a2, ids, wts, s1, s2, z1, z2).cpu().double()
    g, u = (x.double() @ parts[0][3].t()).split(I, dim=1)
    h = g * torch.sigmoid(g) * u
    want = h @ parts[1][3].t()
    two = ((h.half().double() @ parts[1][3].t()).half().double() - want).norm()
    assert (got - want).norm() <= 1.05 * two, "%g times two roundings" % ((got - want).norm() / two).item()
