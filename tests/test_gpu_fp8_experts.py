"""GPU: `fused_experts_fp8` and `fused_moe_fp8` against the definition in 64 bits on the CPU."""
import pytest
import torch

from fp8_reference import assert_within, experts, layer
from helpers import randn

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def routing(T, E, K, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]).to(torch.int32) if T else torch.zeros((0, K), dtype=torch.int32)
    return ids, (torch.rand((T, K), generator=g) + 0.1).to(dtype)


def on_gpu(mlk, l1, l2):
    return mlk.pack_layout_a(l1[0].cuda()), mlk.pack_layout_a(l2[0].cuda()), l1[1].cuda(), l2[1].cuda()


def compare(mlk, T, E, K, H, I, dtype, ids=None, wts=None, place=None, experts_held=None, seed=None, std=1.0):
    l1, l2, w1, w2 = layer(experts_held or E, H, I, seed or T + E)
    x = randn((T, H), dtype, std, T)
    r = routing(T, E, K, dtype, T)
    ids, wts = r[0] if ids is None else ids, r[1] if wts is None else wts
    a1, a2, s1, s2 = on_gpu(mlk, l1, l2)
    args = (x.cuda(), a1, a2, ids.cuda(), wts.cuda(), s1, s2)
    m = None if place is None else place.cuda()
    got = mlk.fused_experts_fp8(*args, experts_map=m)
    want, error = experts(x, w1, w2, ids, wts, place)
    # the weight's product and the sum of a token's picks round in fp32
    assert_within(got, want, error + 2.0 ** -20 * want.abs().max(), dtype, "experts")
    assert torch.equal(got, mlk.fused_experts_fp8(*args, experts_map=m))
    return got


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T,E,K,H,I", [(1, 8, 2, 256, 384), (1, 3, 3, 128, 128), (2, 4, 1, 384, 256), (5, 8, 2, 256, 128), (17, 4, 2, 128, 384), (40, 2, 1, 256, 256),
                                       (33, 16, 4, 128, 128), (70, 2, 2, 128, 256), (150, 3, 1, 256, 128), (300, 2, 1, 128, 128)])
def test_experts(mlk, T, E, K, H, I, dtype):
    compare(mlk, T, E, K, H, I, dtype)


def test_many_picks_and_experts(mlk):
    compare(mlk, 9, 200, 32, 128, 128, BF)


@pytest.mark.parametrize("T", [1, 9, 60, 200])
def test_map_and_dropped_picks(mlk, T):
    """Experts on another card, ids outside the router's, tokens without an expert here."""
    E, K = 8, 3
    place = torch.tensor([2, -1, 0, -1, 1, -1, -1, 3], dtype=torch.int32)
    ids, wts = routing(T, E, K, BF, T + 1)
    ids[T // 2] = torch.tensor([1, -1, 99], dtype=torch.int32)
    if T > 4:
        ids[3] = torch.tensor([-5, 2, 1], dtype=torch.int32)
    got = compare(mlk, T, E, K, 128, 256, BF, ids, wts, place, 4)
    assert (got[T // 2] == 0).all()


@pytest.mark.parametrize("T", [1, 6, 50, 140])
def test_the_same_expert_twice_and_all_on_one(mlk, T):
    ids = torch.zeros((T, 2), dtype=torch.int32)
    ids[:, 0] = 1
    ids[:, 1] = 1
    compare(mlk, T, 3, 2, 128, 128, BF, ids)


@pytest.mark.parametrize("T", [2, 20, 150])
def test_a_token_with_nan_or_infinity_keeps_to_itself(mlk, T):
    l1, l2, _, _ = layer(4, 256, 128, 1)
    a1, a2, s1, s2 = on_gpu(mlk, l1, l2)
    ids, wts = (t.cuda() for t in routing(T, 4, 2, BF, T))
    x = randn((T, 256), BF, 1.0, 2).cuda()
    clean = mlk.fused_experts_fp8(x, a1, a2, ids, wts, s1, s2)
    x[0, 3], x[T - 1, 200] = float("nan"), float("-inf")
    got = mlk.fused_experts_fp8(x, a1, a2, ids, wts, s1, s2)
    assert got[0].isnan().all() and got[-1].isnan().all() and torch.equal(got[1:-1], clean[1:-1])


@pytest.mark.parametrize("T,E,K", [(1, 8, 2), (7, 8, 2), (90, 8, 2), (1100, 8, 2), (2100, 16, 8)])
def test_rows_and_workspace(mlk, T, E, K):
    from muxi_native_layout_kernels_amd import _lib
    lib = _lib.load()
    H, I = 256, 128
    l1, l2, _, _ = layer(E, H, I, T)
    a1, a2, s1, s2 = on_gpu(mlk, l1, l2)
    x = randn((T, H), HF, 1.0, T).cuda()
    ids, wts = (t.cuda() for t in routing(T, E, K, HF, T))
    y = torch.full((T + 8, H), 7.0, dtype=HF, device="cuda")
    need = lib.mlk_experts_fp8_workspace_bytes(T, E, E, K, H, I)
    ws = torch.randint(0, 256, (need + 4096,), dtype=torch.uint8, device="cuda")          # anything
    ws[need:] = 91
    rc = lib.mlk_fused_experts_fp8(a1.data_ptr(), s1.data_ptr(), a2.data_ptr(), s2.data_ptr(), x.data_ptr(), T, E, E, K, H, I, 0, ids.data_ptr(), wts.data_ptr(),
                                   None, y.data_ptr(), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.mlk_last_error()
    assert (y[T:] == 7.0).all() and (ws[need:] == 91).all()
    assert torch.equal(y[:T], mlk.fused_experts_fp8(x, a1, a2, ids, wts, s1, s2))


@pytest.mark.parametrize("T", [1, 30, 200])
def test_graph_replays_and_flat_weights(mlk, T):
    l1, l2, _, _ = layer(4, 256, 128, 1)
    a1, a2, s1, s2 = on_gpu(mlk, l1, l2)
    flat1, flat2 = a1.view(4, 256, 256), a2.view(4, 256, 128)
    ids, wts = (t.cuda() for t in routing(T, 4, 2, BF, T))
    x = randn((T, 256), BF, 1.0, 2).cuda()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        mlk.fused_experts_fp8(x, a1, a2, ids, wts, s1, s2)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = mlk.fused_experts_fp8(x, a1, a2, ids, wts, s1, s2)
    for i in range(4):
        x.copy_(randn((T, 256), BF, 1.0 + i, 10 + i))
        ids.copy_(routing(T, 4, 2, BF, 20 + i)[0])
        graph.replay()
        torch.cuda.synchronize()
        want = mlk.fused_experts_fp8(x, flat1, flat2, ids, wts, s1, s2)
        torch.cuda.synchronize()
        assert torch.equal(out, want)


def test_activations_off_16_bytes_and_empty_batches(mlk):
    l1, l2, _, _ = layer(4, 128, 128, 1)
    a1, a2, s1, s2 = on_gpu(mlk, l1, l2)
    x = randn((9 * 128 + 1,), BF, 1.0, 2).cuda()[1:].view(9, 128)
    ids, wts = (t.cuda() for t in routing(9, 4, 2, BF, 1))
    assert torch.equal(mlk.fused_experts_fp8(x, a1, a2, ids, wts, s1, s2), mlk.fused_experts_fp8(x.clone(), a1, a2, ids, wts, s1, s2))
    assert mlk.fused_experts_fp8(x[:0], a1, a2, ids[:0], wts[:0], s1, s2).shape == (0, 128)


def test_router_products_and_load_together(mlk):
    """As a server runs them: routing with padded tokens, the layer, the load; and `fused_moe_fp8`, which is these calls."""
    from muxi_native_layout_kernels_amd.moe_planC import fused_moe_fp8
    T, E, K, H, I = 40, 16, 4, 256, 128
    l1, l2, w1, w2 = layer(E, H, I, 3)
    a1, a2, s1, s2 = on_gpu(mlk, l1, l2)
    x = randn((T, H), BF, 1.0, 5)
    logits, bias = randn((T, E), BF, 1.0, 6).cuda(), randn((E,), torch.float32, 0.1, 7).cuda()
    mask = torch.arange(T, device="cuda") < 33
    ids, wts = mlk.moe_routing(logits, K, "sigmoid", True, 4, 2, bias, 2.5, mask)
    y = mlk.fused_experts_fp8(x.cuda(), a1, a2, ids, wts, s1, s2)
    want, error = experts(x, w1, w2, ids.cpu(), wts.cpu())
    assert_within(y, want, error + 2.0 ** -20 * want.abs().max(), BF, "layer")
    assert (y[33:] == 0).all()
    load = torch.zeros(E, dtype=torch.int32, device="cuda")
    z = fused_moe_fp8(x.cuda(), a1, a2, logits, K, True, s1, s2, use_grouped_topk=True, num_expert_group=4, topk_group=2, gating_bias=bias, score_func="sigmoid",
                      scaling=2.5, token_mask=mask, expert_load=load)
    assert torch.equal(y, z)
    assert torch.equal(load.cpu(), torch.bincount(ids[:33].cpu().flatten().long(), minlength=E).int())
    assert torch.equal(load, mlk.expert_counts(ids, E))
