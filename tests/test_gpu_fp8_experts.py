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


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("T", [2, 20, 150])
def test_a_token_with_nan_or_infinity_keeps_to_itself(mlk, T, dtype):
    l1, l2, _, _ = layer(4, 256, 128, 1)
    a1, a2, s1, s2 = on_gpu(mlk, l1, l2)
    ids, wts = (t.cuda() for t in routing(T, 4, 2, dtype, T))
    x = randn((T, 256), dtype, 1.0, 2).cuda()
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


def exact_layer(T, E, K, H, I, dtype, held, seed):
    """Arguments of a layer whose every step is exact, and its result: a gate of 32, 64 or 128 for a token, whose SiLU is the gate itself in fp32; up sums of at most 16 products of -1, 0
    and 1, so that an intermediate is a small integer times a power of two, which a code holds; -1, 0 and 1 again in the down projection, whose sums are whole numbers below 2^24; scales
    and weights are powers of two."""
    g = torch.Generator(device="cuda").manual_seed(seed)

    def ints(low, high, shape):
        return torch.randint(low, high, shape, generator=g, device="cuda")

    code = torch.tensor([0xb8, 0, 0x38], dtype=torch.uint8, device="cuda")                    # -1, 0, 1
    w1 = torch.zeros((held, 2 * I, H), dtype=torch.uint8, device="cuda")
    w1[:, :I, 0] = 0x38
    w1[:, I:].scatter_(2, ints(1, H, (held, I, 16)), code[ints(0, 2, (held, I, 16)) * 2])
    w2 = code[ints(0, 3, (held, H, I))]
    s1 = torch.ones((held, 2 * I // 128, H // 128), device="cuda")
    s1[:, I // 128:] = 2.0 ** ints(0, 2, (held, I // 128, 1))
    s2 = 2.0 ** (ints(0, 2, (held, H // 128, I // 128)).float() - (0 if dtype == BF else 10))          # fp16 holds numbers up to 2^16
    x = ints(-1, 2, (T, H)).float()
    x[:, 0] = 2.0 ** ints(5, 8, (T,))
    # some experts are picked far more often than others: tasks of every width
    order = torch.rand((T, E), generator=g, device="cuda") + torch.rand(E, generator=g, device="cuda") * 0.6
    ids = order.topk(K, dim=-1)[1].int()
    wts = 2.0 ** ints(-2, 2, (T, K)).float()
    place = None
    if held < E:
        place = torch.full((E,), -1, dtype=torch.int32, device="cuda")
        place[torch.randperm(E, generator=g, device="cuda")[:held]] = torch.arange(held, dtype=torch.int32, device="cuda")
    y = torch.zeros((T, H), dtype=torch.float64, device="cuda")
    local = ids if place is None else place[ids.long()]
    table = torch.zeros(256, device="cuda")
    table[0xb8], table[0x38] = -1.0, 1.0
    for e in range(held):
        token, pick = (local == e).nonzero(as_tuple=True)
        up = (x[token] @ table[w1[e, I:].int()].t()) * s1[e, I // 128:, 0].repeat_interleave(128)
        h = up * x[token, :1]
        down = table[w2[e].int()] * s2[e].repeat_interleave(128, 0).repeat_interleave(128, 1)
        y.index_add_(0, token, (h.double() @ down.double().t()) * wts[token, pick].double().unsqueeze(1))
    assert y.abs().max() < 2 ** 24
    y = y.to(dtype)
    assert y.isfinite().all()
    return (x.to(dtype), w1, w2, ids, wts.to(dtype), s1, s2, place), y


@pytest.mark.parametrize("T,E,K,H,I,held", [
    (1, 8, 2, 4096, 14336, 8), (1, 16, 12, 256, 14336, 16), (1, 2, 1, 65664, 128, 2), (1, 40, 12, 512, 384, 40), (1, 16, 9, 1024, 256, 5), (2, 8, 2, 4096, 1024, 8), (16, 8, 2, 1152, 2048, 8), (50, 64, 8, 2048, 768, 32),
    (30, 2, 1, 896, 640, 2), (100, 5, 2, 640, 1024, 5), (300, 8, 2, 1024, 8192, 8), (513, 8, 2, 4096, 14336, 8), (700, 3, 1, 640, 1024, 3), (900, 8, 2, 4096, 14336, 3),
    (2048, 8, 2, 4096, 8192, 8), (2500, 16, 8, 256, 384, 16), (1300, 300, 4, 256, 128, 77)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_exact_layers(mlk, T, E, K, H, I, held, dtype):
    """Each plan at sizes where it is taken: one token (also where it or its intermediates do not fit LDS), streamed, panels of every width, the queues, two slices of the down projection, several passes."""
    (x, w1, w2, ids, wts, s1, s2, place), want = exact_layer(T, E, K, H, I, dtype, held, T + E)
    a1, a2 = mlk.pack_layout_a(w1), mlk.pack_layout_a(w2)
    del w1, w2
    got = mlk.fused_experts_fp8(x, a1, a2, ids, wts, s1, s2, experts_map=place)
    assert torch.equal(got, want)
    for n in (1, T // 2, T - 1):                                                              # other plans of the same layer
        if n > 0:
            assert torch.equal(mlk.fused_experts_fp8(x[:n], a1, a2, ids[:n], wts[:n], s1, s2, experts_map=place), want[:n])


@pytest.mark.parametrize("T", [1, 9, 40, 130, 300, 700])
def test_fp16_is_as_good_as_its_rounding(mlk, T):
    """All plans compute gate and up of fp16 layers with exact products, so that codes of the intermediate are those of the definition but for the odd one next to a border: the result is within
    half a step of fp16 in the 2-norm, which is 1.7 times what roundings come to."""
    E, K, H, I = 3, 2, 512, 1024
    l1, l2, w1, w2 = layer(E, H, I, T)
    a1, a2, s1, s2 = on_gpu(mlk, l1, l2)
    ids, wts = routing(T, E, K, HF, T)
    x = randn((T, H), HF, 1.0, T)
    got = mlk.fused_experts_fp8(x.cuda(), a1, a2, ids.cuda(), wts.cuda(), s1, s2).cpu().double()
    want, _ = experts(x, w1, w2, ids, wts)
    assert (got - want).norm() <= 2.0 ** -11 * want.norm()


@pytest.mark.parametrize("T", [1, 30, 200])
def test_two_graphs_of_a_stream_and_eager_calls(mlk, T):
    """They share the stream's workspace, which a layer leaves with whatever it last held."""
    layers = [on_gpu(mlk, *layer(4, 256, 128, s)[:2]) for s in (1, 5)]
    ids, wts = (t.cuda() for t in routing(T, 4, 2, BF, T))
    x = randn((T, 256), BF, 1.0, 2).cuda()

    def run(i):
        a1, a2, s1, s2 = layers[i]
        return mlk.fused_experts_fp8(x, a1, a2, ids, wts, s1, s2)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    with torch.cuda.stream(side):
        run(0)
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], stream=side):
            outs.append(run(i))
    for i in range(3):
        x.copy_(randn((T, 256), BF, 1.0 + i, 10 + i))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            graphs[0].replay()
            eager = run(1)
            graphs[1].replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], run(0)) and torch.equal(outs[1], run(1)) and torch.equal(eager, outs[1])


def test_a_long_batch_leaves_nothing_behind_for_a_short_one(mlk):
    """One workspace, every plan in turn: counters and queues are cleared by the call that uses them."""
    l1, l2, _, _ = layer(8, 256, 256, 9)
    a1, a2, s1, s2 = on_gpu(mlk, l1, l2)
    x = randn((2300, 256), BF, 1.0, 3).cuda()
    ids, wts = (t.cuda() for t in routing(2300, 8, 8, BF, 4))
    alone = {}
    for n in (2300, 1, 40, 7, 300, 2, 2300, 7, 1, 40):
        y = mlk.fused_experts_fp8(x[:n], a1, a2, ids[:n], wts[:n], s1, s2)
        assert torch.equal(y, alone.setdefault(n, y))
