"""GPU: scratch of the e4m3 products and expert layers across calls of different length."""
import pytest
import torch

from fp8_reference import layer
from helpers import randn
from test_gpu_fp8_experts import on_gpu, routing

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.mark.parametrize("dtype", [BF, HF])
def test_scratch_of_the_longest_layer_serves_shorter_ones(mlk, dtype):
    from muxi_native_layout_kernels_amd import _lib
    lib = _lib.load()
    E, K, H, I, most = 8, 2, 256, 8192, 400
    l1, l2, _, _ = layer(E, H, I, 3)
    a1, a2, s1, s2 = on_gpu(mlk, l1, l2)
    x = randn((most, H), dtype, 1.0, 4).cuda()
    ids, wts = (t.cuda() for t in routing(most, E, K, dtype, 5))
    need = lib.mlk_experts_fp8_workspace_bytes(most, E, E, K, H, I)
    ws = torch.randint(0, 256, (need + 4096,), dtype=torch.uint8, device="cuda")
    ws[need:] = 91
    for T in (most, 1, 2, 71, 72, 73, 80, 300):
        y = torch.full((T + 8, H), 7.0, dtype=dtype, device="cuda")
        rc = lib.mlk_fused_experts_fp8(a1.data_ptr(), s1.data_ptr(), a2.data_ptr(), s2.data_ptr(), x.data_ptr(), T, E, E, K, H, I, 0 if dtype == HF else 1, ids.data_ptr(),
                                       wts.data_ptr(), None, y.data_ptr(), ws.data_ptr(), need, torch.cuda.current_stream().cuda_stream)
        assert rc == 0, (T, lib.mlk_last_error())
        assert torch.equal(y[:T], mlk.fused_experts_fp8(x[:T], a1, a2, ids[:T], wts[:T], s1, s2)), T
        assert (y[T:] == 7.0).all() and (ws[need:] == 91).all()


def captured_after_the_longest(mlk, call, most, counts):
    """Eager calls of `most` rows, then a graph of each count on the same stream: the pool hands out no more, and every replay gives what an eager call does."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call(most)
    side.synchronize()
    held = mlk.workspace_bytes_held()
    graphs, outs = [], []
    for n in counts:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            outs.append(call(n))
    assert mlk.workspace_bytes_held() == held
    for _ in range(3):
        for graph, out, n in zip(graphs, outs, counts):
            out.zero_()
            torch.cuda.synchronize()
            with torch.cuda.stream(side):
                graph.replay()
                eager = call(n)
            torch.cuda.synchronize()
            assert torch.equal(out, eager), n


def test_a_shorter_layer_captured_after_the_longest(mlk):
    E, K, H, I, most = 8, 2, 256, 4096, 256
    l1, l2, _, _ = layer(E, H, I, 3)
    a1, a2, s1, s2 = on_gpu(mlk, l1, l2)
    x = randn((most, H), BF, 1.0, 4).cuda()
    ids, wts = (t.cuda() for t in routing(most, E, K, BF, 5))
    captured_after_the_longest(mlk, lambda n: mlk.fused_experts_fp8(x[:n], a1, a2, ids[:n], wts[:n], s1, s2), most, (72, 1, 40, 80))


@pytest.mark.parametrize("n,k", [(8192, 8192), (528, 4096), (2064, 7168)])
def test_scratch_of_the_longest_product_serves_shorter_ones(mlk, n, k):
    from muxi_native_layout_kernels_amd import _lib
    lib = _lib.load()
    A, S = products(mlk, n, k)
    most = 700
    x = randn((most, k), BF, 1.0, 4).cuda()
    need = lib.mlk_gemm_fp8_workspace_bytes(most, n, k, 1)
    ws = torch.zeros(need + 4096, dtype=torch.uint8, device="cuda")
    ws[need:] = 91
    for T in (most, 1, 3, 20, 33, 64, 65, 128, 129, 200, 256, 300):
        c = torch.full((T + 8, n), 7.0, dtype=BF, device="cuda")
        rc = lib.mlk_gemm_layout_a_fp8(A.data_ptr(), S.data_ptr(), x.data_ptr(), 1, None, 0, 0, c.data_ptr(), 1, T, n, k, 1.0, None, ws.data_ptr(), need,
                                       torch.cuda.current_stream().cuda_stream)
        assert rc == 0, (T, lib.mlk_last_error())
        assert torch.equal(c[:T], mlk.gemm_layoutA_fp8(A, S, x[:T])), T
        assert (c[T:] == 7.0).all() and (ws[need:] == 91).all() and (ws[:lib.mlk_gemm_counter_bytes()] == 0).all()


def products(mlk, n, k):
    g = torch.Generator(device="cuda").manual_seed(n + k)
    codes = (torch.randn((n, k), generator=g, device="cuda") * 40).clamp_(-448, 448).to(torch.float8_e4m3fn)
    return mlk.pack_layout_a(codes), torch.rand(((n + 127) // 128, k // 128), generator=g, device="cuda") * 1e-3 + 1e-4


def test_a_shorter_product_captured_after_the_longest(mlk):
    n, k, most = 8192, 8192, 129
    A, S = products(mlk, n, k)
    x = randn((most, k), BF, 1.0, 4).cuda()
    captured_after_the_longest(mlk, lambda t: mlk.gemm_layoutA_fp8(A, S, x[:t]), most, (128, 1, 64, 16))
