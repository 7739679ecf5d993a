"""GPU: `quantize_fp8` and `gemm_layoutA_fp8` against their definitions in 64 bits on the CPU."""
import pytest
import torch

from fp8_reference import F8, assert_within, product_error, quantized, rounded, weights
from helpers import randn

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


def check_quantized(mlk, x):
    """Codes and scales bit for bit: powers of two lose nothing on the way."""
    codes, scales = mlk.quantize_fp8(x.cuda())
    want, s = quantized(x)
    assert codes.dtype == F8 and codes.shape == x.shape and scales.dtype == F32 and tuple(scales.shape) == tuple(s.shape)
    assert torch.equal(scales.cpu().double(), s)
    got = codes.cpu().double()
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(), want.nan_to_num())


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("shape", [(1, 128), (1, 7168), (3, 384), (17, 640), (33, 4736), (1000, 256), (2, 5, 1152), (128,)])
def test_quantize(mlk, shape, dtype):
    g = torch.Generator().manual_seed(sum(shape))
    x = (torch.randn(shape, generator=g) * torch.exp(3 * torch.randn(shape[-1], generator=g))).to(dtype)
    check_quantized(mlk, x)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_quantize_every_number(mlk, dtype):
    """All 65536 patterns (infinities and NaN among them), each as the largest of its block, beside one that is, and below others."""
    every = torch.arange(65536, dtype=torch.int32).to(torch.int16).view(dtype)
    x = torch.zeros(65536, 128, dtype=dtype)
    x[:, 3] = every
    x[:, 77] = every.flip(0)
    check_quantized(mlk, x)
    check_quantized(mlk, every.view(512, 128))
    check_quantized(mlk, every.view(128, 512).t().contiguous().view(512, 128))


def test_quantize_fp32_borders(mlk):
    """Maxima around 448 times powers of two, ties of codes, subnormal, largest and tiny numbers."""
    exact = 448.0 * 2.0 ** torch.arange(-140, 120).double()
    rows = torch.stack([exact.float(), torch.nextafter(exact.float(), torch.tensor(3.4e38)), torch.nextafter(exact.float(), torch.tensor(0.0))], dim=1).flatten()
    x = torch.zeros(rows.numel(), 128)
    x[:, 5] = rows
    tie = torch.arange(-127, 1).float() / 16 + 1.0 / 32                     # halfway between codes
    x += torch.where(torch.arange(128) == 5, 0.0, tie * 0.25) * (rows / 448).unsqueeze(1)
    check_quantized(mlk, x)
    check_quantized(mlk, torch.tensor([[1e-45, -1e-45] + [0.0] * 126, [torch.finfo(F32).max, -1.0] + [1e30] * 126, [0.0] * 128, [-0.0] * 128,
                                       [float("nan")] * 128, [float("inf"), float("-inf")] + [1.0] * 126]))


def test_quantize_calls(mlk):
    x = randn((5, 256), BF, 1.0, 1).cuda()
    flat = randn((5 * 256 + 1,), BF, 1.0, 2).cuda()
    off = flat[1:].view(5, 256)
    assert off.data_ptr() % 16
    a, b = mlk.quantize_fp8(off), mlk.quantize_fp8(off.clone())
    assert torch.equal(a[0].view(torch.uint8), b[0].view(torch.uint8)) and torch.equal(a[1], b[1])
    empty = mlk.quantize_fp8(x[:0])
    assert empty[0].shape == (0, 256) and empty[1].shape == (0, 2)
    with pytest.raises(RuntimeError, match="contiguous"):
        mlk.quantize_fp8(randn((256, 256), BF, 1.0, 1).cuda().t())
    leaf = x.clone().requires_grad_(True)
    assert not mlk.quantize_fp8(leaf)[1].requires_grad


PRODUCTS = [(1, 16, 128), (1, 512, 2048), (2, 48, 384), (5, 272, 1280), (15, 128, 256), (16, 2064, 640), (17, 144, 1152), (31, 528, 384), (48, 272, 640), (64, 528, 1152),
            (65, 272, 1152), (100, 528, 640), (129, 16, 256), (130, 1040, 384), (257, 272, 896), (300, 784, 128)]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("tokens,n,k", PRODUCTS)
def test_product(mlk, tokens, n, k, dtype):
    codes, s, w = weights(n, k, tokens + n)
    x = randn((tokens, k), dtype, 1.0, n + k)
    bias = randn((1, n), dtype, 1.0, 3) if n % 32 == 0 else None
    A, S = mlk.pack_layout_a(codes.cuda()), s.cuda()
    got = mlk.gemm_layoutA_fp8(A, S, x.cuda(), alpha=0.75, bias=None if bias is None else bias.cuda())
    xq = rounded(x)
    want = 0.75 * (xq @ w.t()) + (0.0 if bias is None else bias.double())
    assert got.dtype == dtype
    # alpha and the bias round once each in fp32
    assert_within(got, want, 0.75 * product_error(xq, w) + 2.0 ** -23 * (want.abs() + 4), dtype, "product")
    assert torch.equal(got, mlk.gemm_layoutA_fp8(A, S, x.cuda(), alpha=0.75, bias=None if bias is None else bias.cuda()))


@pytest.mark.parametrize("tokens,n,k", [(1, 144, 640), (7, 272, 384), (40, 272, 640), (130, 528, 384)])
def test_codes_with_scales_of_any_value_and_strides(mlk, tokens, n, k):
    codes, s, w = weights(n, k, tokens)
    g = torch.Generator().manual_seed(n)
    q = (torch.randn((tokens, k), generator=g) * 60).clamp_(-448, 448).to(F8)
    a = torch.randn((tokens, k // 128), generator=g) * 0.02
    xq = q.double() * a.double().repeat_interleave(128, dim=-1)
    A, S, B = mlk.pack_layout_a(codes.cuda()), s.cuda(), q.cuda()
    wide = torch.zeros((tokens, 3 * (k // 128)), device="cuda")
    wide[:, 1::3] = a.cuda()
    for scale in (a.cuda(), a.cuda().t().contiguous().t(), wide[:, 1::3]):
        for dtype in (None, BF, HF):
            got = mlk.gemm_layoutA_fp8(A, S, B, scale, out_dtype=dtype)
            assert got.dtype == (dtype or BF)
            assert_within(got, xq @ w.t(), product_error(xq, w), got.dtype, "codes")
    assert torch.equal(mlk.gemm_layoutA_fp8(A, S, B.view(torch.uint8), a.cuda()), mlk.gemm_layoutA_fp8(A.view(torch.uint8), S, B, a.cuda()))


@pytest.mark.parametrize("tokens", [1, 20, 100, 300])
def test_quantised_ahead_is_the_same(mlk, tokens):
    """One set of codes for several products, as a layer's projections have them: the sums that quantising in each call gives, perhaps in another order."""
    x = randn((tokens, 640), BF, 1.0, 5).cuda()
    q = mlk.quantize_fp8(x)
    for n in (144, 528):
        codes, s, _ = weights(n, 640, n)
        A = mlk.pack_layout_a(codes.cuda())
        got, want = (mlk.gemm_layoutA_fp8(A, s.cuda(), *v).double() for v in (q, (x,)))
        # five windows in fp32: 2^-21 of the sum of magnitudes at most, and results on two sides of a border come out a whole step, 2^-7, apart
        size = mlk.gemm_layoutA_fp8((A.view(torch.uint8) & 0x7f), s.cuda().abs(), x.abs()).double()
        assert ((got - want).abs() <= 2.0 ** -7 * want.abs() + 2.0 ** -20 * size).all()


@pytest.mark.parametrize("tokens", [1, 9, 40, 300])
def test_exact_sums(mlk, tokens):
    """Codes and scales whose products and sums are whole numbers that every format on the way holds: the result is exact."""
    n, k = 272, 384
    g = torch.Generator().manual_seed(1)
    q, c = torch.randint(-2, 3, (tokens, k), generator=g), torch.randint(-1, 2, (n, k), generator=g)
    c[:, 40:] = 0
    s, a = torch.full((3, 3), 0.25), torch.full((tokens, 3), 4.0)
    got = mlk.gemm_layoutA_fp8(mlk.pack_layout_a(c.to(F8).cuda()), s.cuda(), q.to(F8).cuda(), a.cuda())
    assert torch.equal(got.cpu().double(), (q @ c.t()).double())


@pytest.mark.parametrize("tokens,n,k", [
    (65, 16, 256), (65, 16400, 256), (515, 8208, 256), (1300, 11024, 256), (200, 16400, 256), (4100, 4112, 256), (129, 16400, 256), (257, 16400, 256),
    (390, 16400, 256), (2050, 8208, 256), (1030, 11024, 256), (2050, 16400, 2048), (70, 528, 2048), (150, 528, 4096), (300, 2064, 7168), (1030, 2064, 4096), (700, 8208, 7168), (70, 8208, 7168),
    (150, 11024, 7168), (200, 16400, 7168), (257, 16400, 7168), (2050, 16400, 7168), (3000, 16400, 4096)])
def test_exact_sums_in_panels_of_every_shape(mlk, tokens, n, k):
    """Likewise with powers of two as scales, another one for every block, in panels of 128 and 256 rows x 64 to 256 tokens: whole, in slices of k, dealt, in several rounds."""
    g = torch.Generator(device="cuda").manual_seed(tokens)
    q = torch.randint(-2, 3, (tokens, k), generator=g, device="cuda")
    c = torch.randint(-1, 2, (n, k), generator=g, device="cuda")
    s = torch.randint(0, 2, ((n + 127) // 128, k // 128), generator=g, device="cuda").float().exp2()
    a = torch.randint(0, 2, (tokens, k // 128), generator=g, device="cuda").float().exp2()
    got = mlk.gemm_layoutA_fp8(mlk.pack_layout_a(c.to(F8)), s, q.to(F8), a)
    want = (q * a.repeat_interleave(128, 1)) @ (c * s.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)).t()          # fp32, below 2^24
    assert torch.equal(got, want.to(BF))


@pytest.mark.parametrize("k", [512, 2176, 4224, 4608, 12416])
@pytest.mark.parametrize("n", [160, 1040, 1616, 3216, 4816, 7696, 9616, 17616, 26000])
def test_exact_sums_of_every_streaming_launch(mlk, n, k):
    """Likewise through few tokens: rows for a quarter of the CUs' workgroups to more than four each, k whole and in slices, tokens in LDS and not, quantised in the call and ahead of it."""
    g = torch.Generator(device="cuda").manual_seed(n + k)
    c = torch.randint(-1, 2, (n, k), generator=g, device="cuda")
    s = torch.randint(0, 2, ((n + 127) // 128, k // 128), generator=g, device="cuda").float().exp2()
    w = (c * s.repeat_interleave(128, 0)[:n].repeat_interleave(128, 1)).t()
    A = mlk.pack_layout_a(c.to(F8))
    for tokens in (1, 2, 3, 4, 5, 7, 16, 17, 24, 32, 33, 48, 64, 65, 100, 128, 129, 200, 256):
        x = torch.randint(-2, 3, (tokens, k), generator=g, device="cuda").to(BF)
        bias = torch.randint(-9, 10, (1, n), generator=g, device="cuda").to(BF)
        want = (x.float() @ w + bias.float()).to(BF)
        assert torch.equal(mlk.gemm_layoutA_fp8(A, s, x, bias=bias), want), tokens
        assert torch.equal(mlk.gemm_layoutA_fp8(A, s, *mlk.quantize_fp8(x), bias=bias), want), tokens


@pytest.mark.parametrize("tokens", [2, 9, 20, 40, 300])
def test_a_row_with_nan_or_infinity_keeps_to_itself(mlk, tokens):
    codes, s, _ = weights(528, 1024, 1)
    A, S = mlk.pack_layout_a(codes.cuda()), s.cuda()
    x = randn((tokens, 1024), BF, 1.0, 2).cuda()
    clean = mlk.gemm_layoutA_fp8(A, S, x)
    x[0, 5], x[tokens - 1, 1023] = float("nan"), float("inf")
    got = mlk.gemm_layoutA_fp8(A, S, x)
    assert got[0].isnan().all() and got[-1].isnan().all() and torch.equal(got[1:-1], clean[1:-1])


@pytest.mark.parametrize("tokens", [1, 9, 20, 40, 300])
def test_activations_off_16_bytes_and_empty_batches(mlk, tokens):
    codes, s, _ = weights(272, 640, 1)
    A, S = mlk.pack_layout_a(codes.cuda()), s.cuda()
    off = randn((tokens * 640 + 1,), HF, 1.0, 2).cuda()[1:].view(tokens, 640)
    assert off.data_ptr() % 16
    assert torch.equal(mlk.gemm_layoutA_fp8(A, S, off), mlk.gemm_layoutA_fp8(A, S, off.clone()))
    q, a = mlk.quantize_fp8(off)
    raw = torch.empty(tokens * 640 + 3, dtype=torch.uint8, device="cuda")
    raw[3:] = q.view(torch.uint8).flatten()
    # codes against codes: from 16 bits the sums may be taken in another order
    assert torch.equal(mlk.gemm_layoutA_fp8(A, S, raw[3:].view(tokens, 640), a, out_dtype=HF), mlk.gemm_layoutA_fp8(A, S, q, a, out_dtype=HF))
    assert mlk.gemm_layoutA_fp8(A, S, off[:0]).shape == (0, 272)
    assert mlk.gemm_layoutA_fp8(A, S, q[:0], a[:0]).shape == (0, 272)


@pytest.mark.parametrize("tokens,n,k", [(1, 512, 2048), (17, 512, 4096), (50, 272, 640), (65, 272, 1152), (250, 528, 2560), (515, 2064, 1024), (1030, 1040, 384)])
def test_rows_behind_the_last_one_are_left(mlk, tokens, n, k):
    from muxi_native_layout_kernels_amd import _lib
    lib = _lib.load()
    codes, s, _ = weights(n, k, 1)
    A, S, x = mlk.pack_layout_a(codes.cuda()), s.cuda(), randn((tokens, k), BF, 1.0, 2).cuda()
    c = torch.full((tokens + 8, n), 7.0, dtype=BF, device="cuda")
    need = lib.mlk_gemm_fp8_workspace_bytes(tokens, n, k, 1)
    ws = torch.zeros(need + 4096, dtype=torch.uint8, device="cuda")
    ws[need:] = 91
    rc = lib.mlk_gemm_layout_a_fp8(A.data_ptr(), S.data_ptr(), x.data_ptr(), 1, None, 0, 0, c.data_ptr(), 1, tokens, n, k, 1.0, None, ws.data_ptr(), need,
                                   torch.cuda.current_stream().cuda_stream)
    assert rc == 0, lib.mlk_last_error()
    assert torch.equal(c[:tokens], mlk.gemm_layoutA_fp8(A, S, x)) and (c[tokens:] == 7.0).all() and (ws[need:] == 91).all()
    if need:
        assert (ws[:lib.mlk_gemm_counter_bytes()] == 0).all()


@pytest.mark.parametrize("tokens", [1, 9, 20, 40, 300])
def test_graph_replays(mlk, tokens):
    codes, s, _ = weights(528, 640, 1)
    A, S, x = mlk.pack_layout_a(codes.cuda()), s.cuda(), randn((tokens, 640), BF, 1.0, 2).cuda()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        mlk.gemm_layoutA_fp8(A, S, x)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = mlk.gemm_layoutA_fp8(A, S, x)
        codes2, scales2 = mlk.quantize_fp8(x)
    for i in range(4):
        x.copy_(randn((tokens, 640), BF, 1.0 + i, 10 + i))
        graph.replay()
        torch.cuda.synchronize()
        want = mlk.gemm_layoutA_fp8(A, S, x)
        q = mlk.quantize_fp8(x)
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(codes2.view(torch.uint8), q[0].view(torch.uint8)) and torch.equal(scales2, q[1])


def test_streams_side_by_side(mlk):
    codes, s, _ = weights(2064, 2048, 1)
    A, S = mlk.pack_layout_a(codes.cuda()), s.cuda()
    xs = [randn((t, 2048), BF, 1.0, t).cuda() for t in (1, 20, 100, 300)]
    want = [mlk.gemm_layoutA_fp8(A, S, x) for x in xs]
    streams = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = [[] for _ in xs]
    for _ in range(5):
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got[i].append(mlk.gemm_layoutA_fp8(A, S, xs[i]))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        assert all(torch.equal(v, w) for v in g)


def test_offsets_past_32_bits(mlk):
    """Weights of more than 4 GiB, and an output of more than 2^32 elements; a few rows are checked against the same product alone."""
    n, k = 262160, 16512
    g = torch.Generator(device="cuda").manual_seed(1)
    A = torch.randint(0, 120, (n // 16, k // 8, 16, 8), generator=g, device="cuda", dtype=torch.uint8)         # finite codes
    S = torch.rand((n + 127) // 128, k // 128, generator=g, device="cuda") + 0.5
    x = (torch.randn((16400, k), generator=g, device="cuda") * 1e-3).to(BF)
    for tokens in (1, 20, 16400):
        got = mlk.gemm_layoutA_fp8(A, S, x[:tokens])
        # the last two row groups lie in two blocks of scales
        alone = lambda v: torch.cat([mlk.gemm_layoutA_fp8(A[-2:-1].clone(), S[-2:-1].clone(), v), mlk.gemm_layoutA_fp8(A[-1:].clone(), S[-1:].clone(), v)], dim=1)
        last = alone(x[:tokens])
        # the same sums, perhaps in another order: 2^-14 of the sum of magnitudes (all weights are positive, so it is that of |x|), and both are rounded, by at most
            # 2^-8 of themselves each: sums on two sides of a border come out a whole step apart
        tol = alone(x[:tokens].abs()).float() * 2.0 ** -14 + 2.0 ** -7 * last.float().abs()
        assert ((got[:, -32:].float() - last.float()).abs() <= tol).all()
        del got


@pytest.mark.parametrize("tokens", [300, 1 << 21])
def test_scales_far_apart(mlk, tokens):
    """A step from block to block that 32 bits do not hold (here of a single block, so that nothing lies there) leaves the panels, whose offsets of scales are 32 bits."""
    g = torch.Generator(device="cuda").manual_seed(3)
    A = torch.randint(0, 120, (2, 16, 16, 8), generator=g, device="cuda", dtype=torch.uint8)
    S, a = torch.rand((1, 1), generator=g, device="cuda") + 0.5, torch.rand((tokens, 1), generator=g, device="cuda")
    q = torch.randint(0, 120, (tokens, 128), generator=g, device="cuda", dtype=torch.uint8)
    far = a.as_strided((tokens, 1), (1, 1 << 30))
    assert torch.equal(mlk.gemm_layoutA_fp8(A, S, q, far), mlk.gemm_layoutA_fp8(A, S, q, a))


def test_calls_from_a_backward_pass_and_under_grad(mlk):
    """The products are detached: they neither record nor stop a graph around them."""
    codes, s, _ = weights(144, 256, 1)
    A, S = mlk.pack_layout_a(codes.cuda()), s.cuda()
    x = randn((3, 256), BF, 1.0, 1).cuda().requires_grad_(True)
    y = mlk.gemm_layoutA_fp8(A, S, x)
    q, a = mlk.quantize_fp8(x)
    assert not y.requires_grad and not a.requires_grad and not q.requires_grad
    (x.float().sum() + y.float().sum()).backward()
    assert (x.grad == 1).all()
