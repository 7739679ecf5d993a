"""GPU: how the 4-bit products, their expert layers, the balance loss and the expert counts are called: every launch plan, captured graphs, streams, alignment,
long offsets, rows behind the last one."""
import pytest
import torch

from helpers import randn
from test_gpu_w4 import assert_within, on_gpu, term_size, w4_weights
from test_gpu_w4_experts import check as check_experts
from test_gpu_w4_experts import expected as expected_experts
from test_gpu_w4_experts import layer, routing

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("tokens,n,k,group,zeros,dtype", [
    (1, 8208, 256, 64, True, BF), (3, 8208, 256, 64, False, HF), (1, 16400, 128, 32, False, BF), (1, 32, 70016, 128, True, HF), (2, 32, 70016, 128, False, BF),
    (5, 2064, 7168, 128, False, HF), (20, 2064, 7168, 32, True, BF), (37, 2064, 2560, 64, True, HF), (60, 2064, 7168, 3584, False, BF), (40, 8208, 256, 32, True, HF),
    (1, 16, 1280, 640, False, HF), (2050, 272, 7168, 128, True, BF), (1025, 4112, 384, 128, False, HF), (1025, 4112, 512, 32, True, BF),
    (2050, 2064, 2048, 64, False, BF), (300, 528, 2048, 64, True, HF), (129, 16, 256, 32, False, HF)])
def test_every_plan_against_64_bits(mlk, tokens, n, k, group, zeros, dtype):
    codes, s, z, w = w4_weights(n, k, group, dtype, zeros, tokens + n)
    x = randn((tokens, k), dtype, 1.0, 3)
    A, S, Z = mlk.pack_layout_a_w4(*on_gpu(codes, s, z))
    got = mlk.gemm_layoutA_w4(A, S, x.cuda(), Z)
    assert_within(got, x.double() @ w.t(), term_size(x, s, group), dtype, k, "product")
    again = mlk.gemm_layoutA_w4(A, S, x.cuda(), Z)
    assert torch.equal(got, again)                       # no sum's order depends on which workgroup comes first


@pytest.mark.parametrize("tokens", [1, 20, 40, 100, 600])
@pytest.mark.parametrize("dtype", [HF, BF])
def test_extreme_weights_and_activations(mlk, tokens, dtype):
    """Codes and zero points at their ends, scales of zero, subnormal and large, activations of one sign (the offset of the codes cancels most)."""
    n, k, group = 272, 1024, 64
    codes, s, z, _ = w4_weights(n, k, group, dtype, True, 5)
    q = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)
    q[:64], z[:32], z[32:64] = 15, 0, 15
    q[64:128], z[64:96], z[96:128] = 0, 0, 15
    s[::7], s[1::7], s[2::7] = 0.0, torch.finfo(dtype).smallest_normal / 4, 3.0
    w = ((q.double().unflatten(-1, (k // group, group)) - z.double().unsqueeze(-1)) * s.double().unsqueeze(-1)).flatten(-2)
    x = randn((tokens, k), dtype, 1.0, 3).abs()
    x[0, 1::2] = 0.0
    A, S, Z = mlk.pack_layout_a_w4(*on_gpu((q[..., 0::2] | (q[..., 1::2] << 4)).contiguous(), s, z))
    got, want = mlk.gemm_layoutA_w4(A, S, x.cuda(), Z, alpha=0.125), 0.125 * (x.double() @ w.t())
    assert want.abs().max() < torch.finfo(dtype).max / 2
    assert_within(got, want, term_size(x, s, group) * 0.125, dtype, k, "product")


@pytest.mark.parametrize("tokens", [2, 40, 300])
def test_a_row_with_nan_or_infinity_keeps_to_itself(mlk, tokens):
    codes, s, z, _ = w4_weights(528, 1024, 128, BF, True, 1)
    A, S, Z = mlk.pack_layout_a_w4(*on_gpu(codes, s, z))
    x = randn((tokens, 1024), BF, 1.0, 2).cuda()
    clean = mlk.gemm_layoutA_w4(A, S, x, Z)
    x[0, 5], x[tokens - 1, 1023] = float("nan"), float("inf")
    got = mlk.gemm_layoutA_w4(A, S, x, Z)
    assert got[0].isnan().all() and got[-1].isnan().all() and torch.equal(got[1:-1], clean[1:-1])


@pytest.mark.parametrize("tokens", [1, 20, 50, 130])
def test_activations_off_16_bytes_and_empty_batches(mlk, tokens):
    codes, s, z, _ = w4_weights(272, 640, 128, HF, False, 1)
    A, S, Z = mlk.pack_layout_a_w4(*on_gpu(codes, s, z))
    flat = randn((tokens * 640 + 1,), HF, 1.0, 2).cuda()
    off = flat[1:].view(tokens, 640)
    assert off.data_ptr() % 16 != 0
    assert torch.equal(mlk.gemm_layoutA_w4(A, S, off, Z), mlk.gemm_layoutA_w4(A, S, off.clone(), Z))
    assert mlk.gemm_layoutA_w4(A, S, off[:0], Z).shape == (0, 272)
    with pytest.raises(RuntimeError, match="contiguous"):
        mlk.gemm_layoutA_w4(A, S, randn((tokens, 1280), HF, 1.0, 2).cuda()[:, ::2])
    with pytest.raises(RuntimeError, match="CUDA"):
        mlk.gemm_layoutA_w4(A, S, off, bias=torch.zeros(1, 272, dtype=HF))
    p1, p2, _, _ = layer(4, 128, 128, 128, HF, False, 3)
    (a1, s1, _), (a2, s2, _) = mlk.pack_layout_a_w4(*on_gpu(*p1)), mlk.pack_layout_a_w4(*on_gpu(*p2))
    x = flat[1:1 + tokens * 128].view(tokens, 128)
    ids, wts = on_gpu(*routing(tokens, 4, 2, HF, 1))
    assert torch.equal(mlk.fused_experts_w4(x, a1, a2, ids, wts, s1, s2), mlk.fused_experts_w4(x.clone(), a1, a2, ids, wts, s1, s2))
    assert mlk.fused_experts_w4(x[:0], a1, a2, ids[:0], wts[:0], s1, s2).shape == (0, 128)


@pytest.mark.parametrize("tokens,n,k", [(1, 512, 2048), (17, 512, 7168), (50, 272, 640), (65, 272, 1152), (100, 512, 7168), (250, 528, 5120), (1030, 1040, 384), (257, 4112, 8192),
                                        (515, 11024, 1024)])
def test_rows_behind_the_last_one_are_left(mlk, tokens, n, k):
    from muxi_native_layout_kernels_amd import _lib
    lib = _lib.load()
    codes, s, _, _ = w4_weights(n, k, 128, BF, False, 1)
    A, S, _ = mlk.pack_layout_a_w4(*on_gpu(codes, s, None))
    x = randn((tokens, k), BF, 1.0, 2).cuda()
    c = torch.full((tokens + 8, n), 7.0, dtype=BF, device="cuda")
    need = lib.mlk_gemm_w4_workspace_bytes(tokens, n, k, 128)
    ws = torch.zeros(need + 4096, dtype=torch.uint8, device="cuda")
    ws[need:] = 91
    rc = lib.mlk_gemm_layout_a_w4(A.data_ptr(), S.data_ptr(), None, x.data_ptr(), c.data_ptr(), tokens, n, k, 128, 1, 1.0, None, ws.data_ptr(), need,
                                  torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.mlk_last_error()
    assert torch.equal(c[:tokens], mlk.gemm_layoutA_w4(A, S, x)) and (c[tokens:] == 7.0).all() and (ws[need:] == 91).all()
    if need:
        assert (ws[:lib.mlk_gemm_counter_bytes()] == 0).all()


@pytest.mark.parametrize("T,E,K", [(1, 8, 2), (7, 8, 2), (90, 8, 2), (1100, 8, 2), (2100, 16, 8)])
def test_experts_keep_to_their_rows_and_workspace(mlk, T, E, K):
    from muxi_native_layout_kernels_amd import _lib
    lib = _lib.load()
    H, I = 256, 128
    p1, p2, w1, w2 = layer(E, H, I, 64, HF, True, T)
    (a1, s1, z1), (a2, s2, z2) = mlk.pack_layout_a_w4(*on_gpu(*p1)), mlk.pack_layout_a_w4(*on_gpu(*p2))
    x = randn((T, H), HF, 1.0, T)
    ids, wts = routing(T, E, K, HF, T)
    xd, idsd, wtsd = on_gpu(x, ids, wts)
    y = torch.full((T + 8, H), 7.0, dtype=HF, device="cuda")
    need = lib.mlk_experts_w4_workspace_bytes(T, E, E, K, H, I, 64)
    ws = torch.randint(0, 256, (need + 4096,), dtype=torch.uint8, device="cuda")          # anything
    ws[need:] = 91
    rc = lib.mlk_fused_experts_w4(a1.data_ptr(), s1.data_ptr(), z1.data_ptr(), a2.data_ptr(), s2.data_ptr(), z2.data_ptr(), xd.data_ptr(), T, E, E, K, H, I, 64, 0,
                                  idsd.data_ptr(), wtsd.data_ptr(), None, y.data_ptr(), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.mlk_last_error()
    assert (y[T:] == 7.0).all() and (ws[need:] == 91).all()
    assert torch.equal(y[:T], mlk.fused_experts_w4(xd, a1, a2, idsd, wtsd, s1, s2, z1, z2))
    check_experts(y[:T], expected_experts(x, w1, w2, p1[1], p2[1], ids, wts), HF, "experts")


@pytest.mark.parametrize("T,E,K,H,I,group,zeros,dtype", [
    (1, 2, 2, 3328, 128, 128, True, BF), (9, 2, 1, 3328, 128, 32, False, HF), (9, 2, 2, 128, 3328, 64, True, BF), (60, 2, 1, 256, 8192, 128, False, BF),
    (150, 2, 2, 128, 8192, 64, True, HF), (1, 2, 2, 65664, 128, 128, False, BF), (3, 2, 1, 128, 65664, 128, True, BF), (33, 200, 32, 128, 128, 128, False, HF)])
def test_experts_of_every_plan(mlk, T, E, K, H, I, group, zeros, dtype):
    p1, p2, w1, w2 = layer(E, H, I, group, dtype, zeros, T)
    x = randn((T, H), dtype, 1.0, T)
    ids, wts = routing(T, E, K, dtype, T)
    (a1, s1, z1), (a2, s2, z2) = mlk.pack_layout_a_w4(*on_gpu(*p1)), mlk.pack_layout_a_w4(*on_gpu(*p2))
    call = lambda: mlk.fused_experts_w4(x.cuda(), a1, a2, ids.cuda(), wts.cuda(), s1, s2, z1, z2)
    got = call()
    check_experts(got, expected_experts(x, w1, w2, p1[1], p2[1], ids, wts), dtype, "experts")
    assert torch.equal(got, call())


def test_offsets_past_32_bits(mlk):
    """Weights of more than 4 GiB, and an output of more than 2^32 elements: any bytes are valid codes, the last rows are unpacked for the reference."""
    g = torch.Generator(device="cuda").manual_seed(1)
    n, k = 1 << 20, 8448
    A = torch.randint(0, 256, (n // 16, k // 128, 64, 16), dtype=torch.uint8, device="cuda", generator=g)
    S = torch.full((n // 16, k // 128, 16, 1), 2.0 ** -9, dtype=BF, device="cuda")
    last = mlk.unpack_layout_a_w4(A[-4:].contiguous(), S[-4:].contiguous())[0].cpu()
    w = (torch.stack((last & 15, last >> 4), dim=-1).flatten(-2).double() - 8) * 2.0 ** -9
    s = torch.full((64, k // 128), 2.0 ** -9, dtype=BF)
    for tokens in (1, 20, 80):
        x = randn((tokens, k), BF, 1.0, tokens)
        got = mlk.gemm_layoutA_w4(A, S, x.cuda())[:, -64:]
        assert_within(got, x.double() @ w.t(), term_size(x, s, 128), BF, k, "last rows")
    # experts: the last of many against it alone
    E, H, I = 256, 4096, 4224
    del A, S
    a1 = torch.randint(0, 256, (E, 2 * I // 16, H // 128, 64, 16), dtype=torch.uint8, device="cuda", generator=g)
    a2 = torch.randint(0, 256, (E, H // 16, I // 128, 64, 16), dtype=torch.uint8, device="cuda", generator=g)
    assert a1.numel() > 1 << 32
    s1 = torch.full((E, 2 * I // 16, H // 128, 16, 1), 2.0 ** -9, dtype=BF, device="cuda")
    s2 = torch.full((E, H // 16, I // 128, 16, 1), 2.0 ** -9, dtype=BF, device="cuda")
    for T in (1, 12):
        x, wts = randn((T, H), BF, 1.0, T).cuda(), torch.ones((T, 1), dtype=BF, device="cuda")
        many = mlk.fused_experts_w4(x, a1, a2, torch.full((T, 1), E - 1, dtype=torch.int32, device="cuda"), wts, s1, s2)
        one = mlk.fused_experts_w4(x, a1[-1:], a2[-1:], torch.zeros((T, 1), dtype=torch.int32, device="cuda"), wts, s1[-1:], s2[-1:])
        assert torch.equal(many, one) and many.abs().sum() > 0
    del a1, a2, s1, s2
    codes, s, _, w = w4_weights(1 << 20, 128, 128, BF, False, 2)
    A, S, _ = mlk.pack_layout_a_w4(*on_gpu(codes, s, None))
    x = randn((4200, 128), BF, 1.0, 3)
    got = mlk.gemm_layoutA_w4(A, S, x.cuda())
    assert got.numel() > 1 << 32
    for rows in (slice(0, 8), slice(4192, 4200)):
        for cols in (slice(0, 64), slice((1 << 20) - 64, 1 << 20)):
            assert_within(got[rows, cols], x[rows].double() @ w[cols].t(), term_size(x[rows], s[cols], 128), BF, 128, "corner")


def test_two_streams_at_once(mlk):
    """Calls that share K between workgroups, experts and balance losses on two streams side by side give what they give alone."""
    codes, s, z, _ = w4_weights(1024, 7168, 128, BF, True, 1)
    A, S, Z = mlk.pack_layout_a_w4(*on_gpu(codes, s, z))
    p1, p2, _, _ = layer(8, 256, 256, 128, BF, True, 2)
    (a1, s1, z1), (a2, s2, z2) = mlk.pack_layout_a_w4(*on_gpu(*p1)), mlk.pack_layout_a_w4(*on_gpu(*p2))
    jobs = []
    for T in (16, 200):
        x, x2 = randn((T, 7168), BF, 1.0, T).cuda(), randn((T, 256), BF, 1.0, T).cuda()
        ids, wts = on_gpu(*routing(T, 8, 2, BF, T))
        logits = randn((T, 8), BF, 1.0, T).cuda()
        jobs.append(lambda x=x, x2=x2, ids=ids, wts=wts, logits=logits: (
            mlk.gemm_layoutA_w4(A, S, x, Z), mlk.fused_experts_w4(x2, a1, a2, ids, wts, s1, s2, z1, z2), mlk.moe_balance_loss(logits, ids)[0], mlk.expert_counts(ids, 8)))
    want = [job() for job in jobs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in jobs]
    got = [[] for _ in jobs]
    for _ in range(20):
        for st, job, out in zip(streams, jobs, got):
            with torch.cuda.stream(st):
                out.append(job())
    torch.cuda.synchronize()
    for out, ref in zip(got, want):
        for one in out:
            assert all(torch.equal(a, b) for a, b in zip(one, ref))


def replays(run, inputs, fresh):
    """Captures run() on a stream of its own, replays it on three further inputs with eager calls in between, checks every replay against the eager result."""
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(st):
        run()                                            # every shape once: the capture allocates no workspace
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        out = run()
    for i in range(4):
        for t, v in zip(inputs, fresh(i)):
            t.data.copy_(v)
        want = [t.clone() for t in run()]                # eager, on the default stream
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, want)), i
        run()
        torch.cuda.synchronize()


@pytest.mark.parametrize("tokens", [1, 16, 50, 100, 2050])
def test_products_in_a_graph(mlk, tokens):
    codes, s, z, _ = w4_weights(272, 7168, 128, HF, True, 1)
    A, S, Z = mlk.pack_layout_a_w4(*on_gpu(codes, s, z))
    x = randn((tokens, 7168), HF, 1.0, 0).cuda()
    replays(lambda: [mlk.gemm_layoutA_w4(A, S, x, Z)], [x], lambda i: [randn((tokens, 7168), HF, 1.0, i + 1)])


@pytest.mark.parametrize("T", [1, 20, 300, 2100])
def test_router_experts_and_counts_in_a_graph(mlk, T):
    from muxi_layout_kernels.muxi_moe_planC import fused_moe_w4
    E, K, H, I = 16, 8, 256, 256
    p1, p2, _, _ = layer(E, H, I, 128, BF, True, 2)
    (a1, s1, z1), (a2, s2, z2) = mlk.pack_layout_a_w4(*on_gpu(*p1)), mlk.pack_layout_a_w4(*on_gpu(*p2))
    x, logits = randn((T, H), BF, 1.0, 0).cuda(), randn((T, E), BF, 1.0, 1).cuda()
    load = torch.zeros(E, dtype=torch.int32, device="cuda")

    def run():
        before = load.clone()
        y = fused_moe_w4(x, a1, a2, logits, K, True, s1, s2, z1, z2, expert_load=load)
        return [y, load - before]
    replays(run, [x, logits], lambda i: [randn((T, H), BF, 1.0, i + 2), randn((T, E), BF, 1.0, i + 9)])


@pytest.mark.parametrize("sequences", [None, 5, 100])
def test_balance_loss_and_gradient_in_a_graph(mlk, sequences):
    """Forward and backward; the leaf's eager losses are dropped before the capture, and while it runs."""
    T, E, K = 3000, 64, 6
    logits = randn((T, E), BF, 1.0, 0).cuda().requires_grad_(True)
    ids = torch.randint(0, E, (T, K), dtype=torch.int32, device="cuda")
    cu = None if sequences is None else torch.linspace(0, T, sequences + 1).int().cuda()
    up = torch.tensor(3.0, device="cuda")

    def run():
        loss, counts = mlk.moe_balance_loss(logits, ids, cu_seqlens=cu)
        grad, = torch.autograd.grad(loss, logits, grad_outputs=up)
        return [loss.detach(), counts, grad]
    g = torch.Generator().manual_seed(3)
    replays(run, [logits, ids], lambda i: [randn((T, E), BF, 1.0, i + 1), torch.randint(0, E, (T, K), dtype=torch.int32, generator=g)])


def test_counts_in_a_graph(mlk):
    for T, E in ((64, 256), (30000, 64)):
        ids = torch.randint(0, E, (T, 6), dtype=torch.int32, device="cuda")
        replays(lambda: [mlk.expert_counts(ids, E)], [ids], lambda i: [torch.randint(0, E, (T, 6), dtype=torch.int32)])


@pytest.mark.parametrize("dtype", [HF, BF, torch.float32])
@pytest.mark.parametrize("E", [8, 64, 256])
def test_logits_off_their_vectors(mlk, dtype, E):
    """A view that begins one element on: the loss, the counts and the gradient are those of its copy."""
    T, K = 333, 4
    flat = randn((T * E + 1,), dtype, 1.0, E).cuda()
    ids = torch.randint(0, E, (T, K), dtype=torch.int32, device="cuda")
    out = []
    for view in (flat[1:].view(T, E), flat[1:].clone().view(T, E)):
        leaf = view.detach().requires_grad_(True)
        loss, counts = mlk.moe_balance_loss(leaf, ids, "sigmoid")
        out.append((loss.detach(), counts, torch.autograd.grad(loss, leaf)[0]))
    assert all(torch.equal(a, b) for a, b in zip(*out))


def test_workspaces_are_counted_and_released(mlk):
    logits, ids = torch.randn(5000, 64, device="cuda"), torch.zeros((5000, 2), dtype=torch.int32, device="cuda")
    before = mlk.moe_balance_loss(logits, ids)[0]
    torch.cuda.synchronize()
    assert mlk.ops.workspace_bytes_held() > 0
    assert mlk.ops.release_workspaces() > 0 and mlk.ops.workspace_bytes_held() == 0
    assert torch.equal(mlk.moe_balance_loss(logits, ids)[0], before)


def test_a_refused_layer_counts_nothing(mlk):
    from muxi_layout_kernels.muxi_moe_planC import fused_moe_w4
    p1, p2, _, _ = layer(4, 128, 128, 128, BF, True, 1)
    (a1, s1, z1), (a2, s2, z2) = mlk.pack_layout_a_w4(*on_gpu(*p1)), mlk.pack_layout_a_w4(*on_gpu(*p2))
    load = torch.zeros(4, dtype=torch.int32, device="cuda")
    x, logits = randn((3, 128), BF, 1.0, 1).cuda(), randn((3, 4), BF, 1.0, 2).cuda()
    with pytest.raises(RuntimeError, match="both w1 and w2"):
        fused_moe_w4(x, a1, a2, logits, 2, True, s1, s2, z1, None, expert_load=load)
    with pytest.raises(RuntimeError, match="n_experts"):
        fused_moe_w4(x, a1, a2, logits, 2, True, s1, s2, z1, z2, expert_load=load[:3])
    assert (load == 0).all()
    fused_moe_w4(x, a1, a2, logits, 2, True, s1, s2, z1, z2, expert_load=load)
    assert load.sum() == 6


def packed_at_random(n, k, group, zeros, dtype, seed):
    """Weights in the layout on the GPU: any bytes are valid codes."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    shape = (n // 16, k // max(128, group), 16, max(1, 128 // group))
    A = torch.randint(0, 256, (n // 16, k // 128, 64, 16), dtype=torch.uint8, device="cuda", generator=g)
    S = ((torch.rand(shape, device="cuda", generator=g) + 0.5) * (k ** -0.5 / 4.6)).to(dtype)
    Z = torch.randint(0, 16, shape, dtype=torch.uint8, device="cuda", generator=g) if zeros else None
    return A, S, Z


def check_some_rows(mlk, A, S, Z, group, x, bias, got):
    """Nine row groups at the start, in the middle and at the end against 64 bits."""
    k, groups = x.shape[1], A.shape[0]
    for first in (0, groups // 2 - 3, groups - 9):
        rows, cols = slice(first, first + 9), slice(first * 16, (first + 9) * 16)
        codes, s, z = mlk.unpack_layout_a_w4(A[rows].contiguous(), S[rows].contiguous(), None if Z is None else Z[rows].contiguous())
        q = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).cpu().double()
        off = torch.full(s.shape, 8.0, dtype=torch.float64) if z is None else z.cpu().double()
        w = (q - off.repeat_interleave(group, dim=1)) * s.cpu().double().repeat_interleave(group, dim=1)
        b = bias[:, cols].double()
        assert_within(got[:, cols], x.double() @ w.t() + b, term_size(x, s.cpu(), group) + b.abs(), x.dtype, k, "rows %d" % first)


@pytest.mark.parametrize("n,k,group,zeros,dtype", [(24592, 384, 128, False, BF), (24592, 256, 32, True, HF), (57360, 128, 64, True, BF), (8192, 18432, 128, True, HF),
                                                   (4112, 36864, 32, False, BF)])
@pytest.mark.parametrize("tokens", [5, 16, 20, 33, 48, 49])
def test_eight_row_groups_a_workgroup(mlk, tokens, n, k, group, zeros, dtype):
    A, S, Z = packed_at_random(n, k, group, zeros, dtype, n + tokens)
    x, bias = randn((tokens, k), dtype, 1.0, 3), randn((1, n), dtype, 1.0, 4)
    got = mlk.gemm_layoutA_w4(A, S, x.cuda(), Z, bias=bias.cuda())
    assert torch.equal(got, mlk.gemm_layoutA_w4(A, S, x.cuda(), Z, bias=bias.cuda()))
    check_some_rows(mlk, A, S, Z, group, x, bias, got)


@pytest.mark.parametrize("tokens,n,k,group,zeros,dtype", [
    (257, 11024, 1024, 32, True, HF), (257, 11024, 1024, 64, False, BF), (257, 11024, 1152, 128, True, BF), (515, 11024, 1024, 64, True, HF), (2050, 11024, 1024, 32, False, BF),
    (515, 11024, 1152, 128, False, HF), (130, 4112, 14336, 128, True, BF), (257, 4112, 8192, 64, False, HF), (70, 8208, 14336, 64, True, BF), (70, 11024, 8192, 128, False, BF),
    (257, 8208, 14336, 32, True, BF), (515, 4112, 14336, 32, False, HF), (515, 11024, 1024, 512, True, BF)])
def test_panels(mlk, tokens, n, k, group, zeros, dtype):
    """Panels of 64 and of 128 tokens, whole and in slices of k; the last one holds a single row group."""
    from muxi_native_layout_kernels_amd import _lib
    per = 128 // group if group < 128 else 1
    sums = (tokens * (k // 128 * per + 1) * 16 + 255) // 256 * 256
    need = _lib.load().mlk_gemm_w4_workspace_bytes(tokens, n, k, group) - 65536 - sums
    assert need >= 0 and need % (tokens * n * 4) == 0, "the plan has no panels here: take another size"
    A, S, Z = packed_at_random(n, k, group, zeros, dtype, n + tokens)
    x, bias = randn((tokens, k), dtype, 1.0, 3), randn((1, n), dtype, 1.0, 4)
    got = mlk.gemm_layoutA_w4(A, S, x.cuda(), Z, bias=bias.cuda())
    check_some_rows(mlk, A, S, Z, group, x, bias, got)
    x[3, 7] = float("nan")                               # keeps to its row
    other = mlk.gemm_layoutA_w4(A, S, x.cuda(), Z, bias=bias.cuda())
    assert other[3].isnan().all() and torch.equal(other[4:], got[4:]) and torch.equal(other[:3], got[:3])


@pytest.mark.parametrize("tokens", [300, 1030])
def test_panels_in_a_graph_and_off_16_bytes(mlk, tokens):
    A, S, Z = packed_at_random(11024, 1024, 64, True, BF, 1)
    x = randn((tokens, 1024), BF, 1.0, 0).cuda()
    replays(lambda: [mlk.gemm_layoutA_w4(A, S, x, Z)], [x], lambda i: [randn((tokens, 1024), BF, 1.0, i + 1)])
    off = torch.empty(tokens * 1024 + 1, dtype=BF, device="cuda")[1:].view(tokens, 1024).copy_(x)
    assert off.data_ptr() % 16 and torch.equal(mlk.gemm_layoutA_w4(A, S, off, Z), mlk.gemm_layoutA_w4(A, S, x, Z))


@pytest.mark.parametrize("T,E,K,same", [(2, 3, 1, True), (3, 40, 20, False), (32, 4, 2, False), (33, 4, 2, False), (64, 2, 1, True), (64, 5, 1, False), (7, 200, 9, False)])
def test_few_pairs_and_one_more(mlk, T, E, K, same):
    """Up to 64 pairs the kernels find their tasks by themselves, above an alignment launch does: experts with none, one, 16, 17 and all of the pairs, some dropped."""
    p1, p2, w1, w2 = layer(E, 128, 256, 64, BF, True, T)
    (a1, s1, z1), (a2, s2, z2) = mlk.pack_layout_a_w4(*on_gpu(*p1)), mlk.pack_layout_a_w4(*on_gpu(*p2))
    x = randn((T, 128), BF, 1.0, T)
    ids, wts = routing(T, E, K, BF, T)
    if same:
        ids[:] = E - 1
    ids[T // 2, 0] = -1
    got = mlk.fused_experts_w4(x.cuda(), a1, a2, ids.cuda(), wts.cuda(), s1, s2, z1, z2)
    check_experts(got, expected_experts(x, w1, w2, p1[1], p2[1], ids, wts), BF, "experts")
    gone = torch.full_like(ids, E)
    assert (mlk.fused_experts_w4(x.cuda(), a1, a2, gone.cuda(), wts.cuda(), s1, s2, z1, z2) == 0).all()


@pytest.mark.parametrize("tokens", [1, 20, 100])
def test_subnormal_activations_count(mlk, tokens):
    """fp16 activations below 2^-14 all of them: the results are some hundred times the least number, and off by its half at most."""
    n, k, group = 272, 1024, 128
    codes, s, z, _ = w4_weights(n, k, group, HF, True, 5)
    s = torch.ones_like(s)
    q = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).double()
    w = q - z.double().repeat_interleave(group, dim=1)
    x = (randn((tokens, k), torch.float32, 1.0, 3) * 1e-6).to(HF)
    assert (x.abs() < 2.0 ** -14).all() and (x != 0).any()
    A, S, Z = mlk.pack_layout_a_w4(*on_gpu(codes, s, z))
    assert_within(mlk.gemm_layoutA_w4(A, S, x.cuda(), Z), x.double() @ w.t(), term_size(x, s, group), HF, k, "product")


def test_one_workspace_for_counts_and_losses(mlk):
    """Counts of a long prompt and balance losses in turn on one stream, of different sizes: what one leaves is what the other expects."""
    g = torch.Generator().manual_seed(4)
    for T, E in ((3000, 64), (9000, 256), (1500, 8), (20000, 100)):
        ids = torch.randint(-1, E + 1, (T, 6), generator=g, dtype=torch.int32)
        kept = ids[(ids >= 0) & (ids < E)].long()
        want = torch.bincount(kept, minlength=E).int()
        logits = torch.randn((T, E), generator=g).cuda()
        for _ in range(3):
            assert torch.equal(mlk.expert_counts(ids.cuda(), E).cpu(), want)
            assert torch.equal(mlk.moe_balance_loss(logits, ids.cuda())[1].cpu(), want)


@pytest.mark.parametrize("T,E,K,H,I,group,zeros,dtype", [
    (20, 4, 2, 256, 128, 32, True, BF), (33, 3, 1, 128, 384, 64, False, HF), (77, 6, 3, 640, 128, 128, True, HF), (60, 2, 2, 256, 8192, 64, True, BF), (140, 4, 1, 384, 256, 32, False, HF),
    (150, 8, 4, 128, 128, 128, False, BF)])
def test_experts_of_two_blocks_a_task(mlk, T, E, K, H, I, group, zeros, dtype):
    """9 to 80 pairs an expert: full and half tasks, an expert with none, one with all, dropped pairs."""
    p1, p2, w1, w2 = layer(E, H, I, group, dtype, zeros, T)
    x = randn((T, H), dtype, 1.0, T)
    (a1, s1, z1), (a2, s2, z2) = mlk.pack_layout_a_w4(*on_gpu(*p1)), mlk.pack_layout_a_w4(*on_gpu(*p2))
    for case in range(3):
        ids, wts = routing(T, E, K, dtype, T + case)
        if case == 1:
            ids[ids == 0] = -1                           # nobody's
        if case == 2:
            ids[:, 0] = E - 1
        y = mlk.fused_experts_w4(x.cuda(), a1, a2, ids.cuda(), wts.cuda(), s1, s2, z1, z2)
        check_experts(y, expected_experts(x, w1, w2, p1[1], p2[1], ids, wts), dtype, "experts, routing %d" % case)


@pytest.mark.parametrize("T,E,held,K", [(160, 64, 4, 4), (200, 16, 4, 2), (700, 16, 4, 2), (60, 12, 3, 8)])
@pytest.mark.parametrize("here", ["its share", "all", "none"])
def test_a_share_of_the_experts_whatever_comes(mlk, T, E, held, K, here):
    """Plans expect the held experts' share of the pairs; all of them or none may come."""
    p1, p2, w1, w2 = layer(held, 128, 256, 128, BF, True, T)
    (a1, s1, z1), (a2, s2, z2) = mlk.pack_layout_a_w4(*on_gpu(*p1)), mlk.pack_layout_a_w4(*on_gpu(*p2))
    x = randn((T, 128), BF, 1.0, T)
    ids, wts = routing(T, E, K, BF, T)
    emap = torch.full((E,), -1, dtype=torch.int32)
    emap[:held] = torch.arange(held, dtype=torch.int32)
    if here == "all":
        ids = ids % held
    if here == "none":
        ids = ids % (E - held) + held
    ids = ids.int().contiguous()
    y = mlk.fused_experts_w4(x.cuda(), a1, a2, ids.cuda(), wts.cuda(), s1, s2, z1, z2, experts_map=emap.cuda())
    check_experts(y, expected_experts(x, w1, w2, p1[1], p2[1], ids, wts, emap), BF, "experts here")


def test_a_refused_layer_launches_nothing(mlk, monkeypatch):
    """Whatever is wrong with the experts, the bias or the load is said ahead of the router."""
    from muxi_layout_kernels.muxi_moe_planC import fused_moe_w4
    p1, p2, _, _ = layer(4, 128, 128, 64, BF, True, 1)
    (a1, s1, z1), (a2, s2, z2) = mlk.pack_layout_a_w4(*on_gpu(*p1)), mlk.pack_layout_a_w4(*on_gpu(*p2))
    x, logits = randn((3, 128), BF, 1.0, 1).cuda(), randn((3, 4), BF, 1.0, 2).cuda()
    load, bias = torch.zeros(4, dtype=torch.int32, device="cuda"), torch.zeros(4, dtype=BF, device="cuda")
    launched = []
    real = mlk.ops.fused_routing_gate
    monkeypatch.setattr(mlk.ops, "fused_routing_gate", lambda *a, **k: launched.append(1) or real(*a, **k))

    def off(t, by):                                      # the same, so many bytes past 16
        flat = torch.empty(t.numel() * t.element_size() + 16, dtype=torch.uint8, device="cuda")[by:by + t.numel() * t.element_size()].view(t.dtype)
        return flat.view(t.shape).copy_(t)

    def call(match, w1=a1, w2=a2, s1=s1, s2=s2, z1=z1, z2=z2, **kw):
        with pytest.raises(RuntimeError, match=match):
            fused_moe_w4(x, w1, w2, logits, 2, True, s1, s2, z1, z2, **kw)
        assert not launched, match
    call("both w1 and w2", z2=None)
    call("scales of w2", s2=s2[:, :, :, :8].contiguous())
    call("activation dtype", s1=s1.half(), s2=s2.half())
    call("CUDA", w2=a2.cpu())
    call("contiguous", w1=a1.transpose(-1, -2).contiguous().transpose(-1, -2))
    call("16 bytes", w1=off(a1, 8))
    call("8 bytes", s2=off(s2, 4))
    call("on 4", z1=off(z1, 2))
    call("experts_map", experts_map=torch.zeros(4, dtype=torch.int64, device="cuda"))
    call("n_experts", expert_load=load[:3])
    call("n_experts", expert_load=load.long())
    call("CUDA", expert_load=load.cpu())
    call("contiguous", expert_load=torch.zeros(8, dtype=torch.int32, device="cuda")[::2])
    call("every expert", gating_bias=bias[:3])
    call("device", gating_bias=bias.cpu())
    call("contiguous", gating_bias=torch.zeros(8, dtype=BF, device="cuda")[::2])
    fused_moe_w4(x, a1, a2, logits, 2, True, s1, s2, z1, z2, gating_bias=bias, expert_load=load)
    assert launched == [1] and load.sum() == 6


@pytest.mark.parametrize("group,zeros,dtype", [(128, False, BF), (32, True, HF), (64, True, BF)])
@pytest.mark.parametrize("dropped", [False, True])
def test_one_token_whose_intermediates_pass_128_kib(mlk, group, zeros, dtype, dropped):
    """Eight picks of 8320: the down projection reads them from memory, not from LDS."""
    E, K, H, I = 8, 8, 128, 8320
    assert 2 * K * I > 128 * 1024
    p1, p2, w1, w2 = layer(E, H, I, group, dtype, zeros, 3)
    (a1, s1, z1), (a2, s2, z2) = mlk.pack_layout_a_w4(*on_gpu(*p1)), mlk.pack_layout_a_w4(*on_gpu(*p2))
    x, (ids, wts) = randn((1, H), dtype, 1.0, 5), routing(1, E, K, dtype, 5)
    if dropped:
        ids[0, 3], ids[0, 7] = -1, ids[0, 6]             # nobody's, and one expert twice
    got = mlk.fused_experts_w4(x.cuda(), a1, a2, ids.cuda(), wts.cuda(), s1, s2, z1, z2)
    check_experts(got, expected_experts(x, w1, w2, p1[1], p2[1], ids, wts), dtype, "one token")
    assert torch.equal(got, mlk.fused_experts_w4(x.cuda(), a1, a2, ids.cuda(), wts.cuda(), s1, s2, z1, z2))
    gone = torch.full_like(ids, -1)
    assert (mlk.fused_experts_w4(x.cuda(), a1, a2, gone.cuda(), wts.cuda(), s1, s2, z1, z2) == 0).all()
