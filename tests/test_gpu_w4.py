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
