"""GPU: 4-bit weights with group scales, `pack_layout_a_w4`, `gemm_layoutA_w4` and `gemv_layoutA_w4`, against 64 bits on the CPU."""
import pytest
import torch

from helpers import randn

pytestmark = pytest.mark.gpu


def w4_weights(n, k, group, dtype, zeros, seed, lead=()):
    """Row-major codes, scales and zero points on the CPU and the weights they stand for, in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 16, lead + (n, k), generator=g, dtype=torch.uint8)
    s = ((torch.rand(lead + (n, k // group), generator=g) + 0.5) * (k ** -0.5 / 4.6)).to(dtype)
    s = s * torch.where(torch.rand(s.shape, generator=g) < 0.2, -1.0, 1.0).to(dtype)          # scales may be negative
    z = torch.randint(0, 16, s.shape, generator=g, dtype=torch.uint8) if zeros else None
    off = torch.full(s.shape, 8.0, dtype=torch.float64) if z is None else z.double()
    w = ((q.double().unflatten(-1, (k // group, group)) - off.unsqueeze(-1)) * s.double().unsqueeze(-1)).flatten(-2)
    codes = q[..., 0::2] | (q[..., 1::2] << 4)
    return codes.contiguous(), s, z, w


def on_gpu(*ts):
    return [None if t is None else t.cuda() for t in ts]


def assert_within(got, want, size, dtype, k, what=""):
    """Half a step of the result for its rounding, and the fp32 sums: every step of 32 k rounds twice at most (into the sum of its group,
    into the total), each time by 2^-24 of what has been summed, which is no more than `size` = sum over k of ((16 + q) + (16 + z)) |s x|.  That bounds
    the error by k / 16 2^-24 size; a quarter of it is allowed."""
    err = (got.detach().cpu().double() - want).abs()
    tol = torch.finfo(dtype).eps / 2 * want.abs() * 1.01 + size * (k / 64) * 2.0 ** -24 + 1e-30
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25                                   # half a step of the smallest numbers
    worst = (err - tol).max().item() if err.numel() else 0.0
    assert worst <= 0, "%s: off by %g more than allowed (largest error %g)" % (what, worst, err.max().item())


def term_size(x, s, group):
    """(16 + q) + (16 + z) <= 62."""
    return 62.0 * (x.double().abs() @ s.double().abs().repeat_interleave(group, dim=-1).t())


@pytest.mark.parametrize("lead", [(), (3,)])
@pytest.mark.parametrize("n,k,group", [(16, 128, 32), (48, 384, 64), (32, 1280, 128), (64, 768, 384), (16, 256, 256)])
def test_layout_is_a_permutation_and_unpacks(mlk, n, k, group, lead):
    codes, s, z, _ = w4_weights(n, k, group, torch.float16, True, n + k, lead)
    A, S, Z = mlk.pack_layout_a_w4(*on_gpu(codes, s, z))
    # the layout from its definition
    q = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)                            # [.., n, k]
    want = torch.zeros(lead + (n // 16, k // 128, 64, 16), dtype=torch.uint8)
    qq = q.reshape((-1, n // 16, 16, k // 128, 4, 4, 8))                                     # batch, rg, r, t, j, o, c
    out = want.view(-1, n // 16, k // 128, 4, 16, 4, 4)                                      # batch, rg, t, o, r, j, byte
    lay = qq.permute(0, 1, 3, 5, 2, 4, 6)                                                    # batch, rg, t, o, r, j, c
    nib = torch.empty_like(lay)
    for c in range(8):
        nib[..., c // 2 + 4 * (c % 2)] = lay[..., c]
    out.copy_(nib[..., 0::2] | (nib[..., 1::2] << 4))
    assert torch.equal(A.cpu(), want)
    per = max(1, 128 // group)
    for got, src in ((S, s), (Z, z)):
        assert torch.equal(got.cpu(), src.reshape(lead + (n // 16, 16, k // group // per, per)).transpose(-3, -2))
    back = mlk.unpack_layout_a_w4(A, S, Z)
    for got, src in zip(back, (codes, s, z)):
        assert torch.equal(got.cpu(), src)
    none = mlk.unpack_layout_a_w4(*mlk.pack_layout_a_w4(*on_gpu(codes, s, None)))
    assert none[2] is None and torch.equal(none[0].cpu(), codes)


@pytest.mark.parametrize("tokens", [1, 2, 15, 16, 17, 33, 48, 64, 65, 130, 257])
@pytest.mark.parametrize("n,k,group,zeros,dtype", [
    (16, 128, 32, True, torch.float16), (48, 640, 64, False, torch.bfloat16), (272, 1152, 128, True, torch.bfloat16),
    (4112, 256, 32, False, torch.bfloat16), (512, 7168, 128, False, torch.float16), (96, 1536, 768, True, torch.float16)])
def test_product_against_64_bits(mlk, tokens, n, k, group, zeros, dtype):
    codes, s, z, w = w4_weights(n, k, group, dtype, zeros, tokens + n)
    x, bias = randn((tokens, k), dtype, 1.0, 3), randn((1, n), dtype, 1.0, 4)
    A, S, Z = mlk.pack_layout_a_w4(*on_gpu(codes, s, z))
    want, size = x.double() @ w.t(), term_size(x, s, group)
    got = mlk.gemm_layoutA_w4(A, S, x.cuda(), Z)
    assert got.shape == (tokens, n) and got.dtype == dtype
    assert_within(got, want, size, dtype, k, "product")
    got = mlk.gemm_layoutA_w4(A, S, x.cuda(), Z, alpha=0.5, bias=bias.cuda())
    assert_within(got, 0.5 * want + bias.double(), size + bias.double().abs(), dtype, k, "product with alpha and bias")
    if tokens == 1:
        assert torch.equal(mlk.gemv_layoutA_w4(A, S, x.cuda(), Z, alpha=0.5, bias=bias.cuda()), got)


def centred_weights(n, k, group, zeros, seed):
    """fp16 weights as a quantiser leaves them: codes around their zero point, positive scales.  Row-major parts and the weights in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    s = ((torch.rand((n, k // group), generator=g) + 0.5) * (k ** -0.5 / 2.6)).half()
    z = torch.randint(5, 12, s.shape, generator=g, dtype=torch.uint8) if zeros else None
    off = torch.full(s.shape, 8.0) if z is None else z.float()
    q = (torch.randn((n, k // group, group), generator=g) * 2.6 + off.unsqueeze(-1)).round().clamp(0, 15)
    w = ((q.double() - off.double().unsqueeze(-1)) * s.double().unsqueeze(-1)).flatten(-2)
    q = q.flatten(-2).to(torch.uint8)
    return (q[:, 0::2] | (q[:, 1::2] << 4)).contiguous(), s, z, w


def runs_panels(tokens, n, k, group):
    """The panels' workspace: counters, sums of the activations, partial sums where k is split."""
    from muxi_native_layout_kernels_amd import _lib
    per = 128 // group if group < 128 else 1
    need = _lib.load().mlk_gemm_w4_workspace_bytes(tokens, n, k, group) - 65536 - (tokens * (k // 128 * per + 1) * 16 + 255) // 256 * 256
    return need >= 0 and need % (tokens * n * 4) == 0


@pytest.mark.parametrize("mean", [0.0, 1.0, 20.0])
@pytest.mark.parametrize("tokens,times,k,group,zeros", [(515, 4, 14336, 128, False), (400, 8, 14336, 32, True), (300, 8, 14336, 64, True), (400, 16, 14208, 128, False), (400, 16, 14208, 32, True)])
def test_error_does_not_grow_with_the_mean_of_the_activations(mlk, tokens, times, k, group, zeros, mean):
    """The 2-norm of the error is that of one rounding to fp16, give or take a twentieth, whatever the mean m of the activations and the number of tokens.

    One rounding: 2^-11 / sqrt(3) times 0.72 (numbers spread over a binade), 2.0e-4 of the result; a twentieth more leaves sqrt(1.05^2 - 1) = 0.32 of that, 6.5e-5, to the
    fp32 sums.  The result is 2.6 sqrt(k (1 + m^2)) s, 310 m s and more.  Rounding to nearest adds 2^-24 / sqrt(3) of what is held at every step:
      within a window    k / 16 steps that hold half of 24 * 128 m s on average: sqrt(k / 48) * 1540 / 310 * 2^-24 = 5e-6 of the result
      sums of groups     k / 32 steps at most.  Offsets that are taken out of every group leave nothing; such that cancel between neighbouring windows leave the difference
                         of their scales, 24 * 128 * 0.41 m s, in k / 256 pairs at random: 9400 m s at the end.  sqrt(k / 96) * 9400 / 310 * 2^-24 = 2.2e-5 of the result
    An offset that is held for all of k until the end, 24 k m s, comes to 1.2e-4 of the result, 1.2 roundings."""
    codes, s, z, w = centred_weights(528, k, group, zeros, k + group)
    x = (randn((tokens, k), torch.float32, 1.0, 3) + mean).half()
    A, S, Z = mlk.pack_layout_a_w4(*[None if t is None else t.cuda().repeat(times, 1) for t in (codes, s, z)])
    assert runs_panels(tokens, 528 * times, k, group), "the plan has no panels here: take another size"
    want = x.double() @ w.t()
    for rows in (slice(None), slice(0, 20)):                 # panels; few tokens
        got = mlk.gemm_layoutA_w4(A, S, x[rows].cuda(), Z).cpu().double().unflatten(1, (times, 528)) - want[rows].unsqueeze(1)
        one = (want[rows].half().double() - want[rows]).norm() * times ** 0.5
        assert got.norm() <= 1.05 * one, "%g roundings" % (got.norm() / one).item()
