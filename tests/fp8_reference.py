"""The e4m3 products and expert layers from their definitions in 64 bits on the CPU, and how far the kernels may be from them."""
import torch

F8 = torch.float8_e4m3fn
HALF = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}       # half a step, relative


def e4m3(v):
    """|v| <= 448 rounded to the nearest e4m3 number, ties to even: steps of 2^(exponent - 3), 2^-9 at least."""
    exponent = torch.frexp(v)[1] - 1
    step = torch.ldexp(torch.ones_like(v), exponent.clamp(min=-6) - 3)
    return torch.round(v / step) * step


def block_scales(x):
    """[.., K] in 64 bits -> the smallest power of two, 2^-100 at least, with max |finite x| <= 448 scale, [.., K/128]."""
    most = torch.where(x.isfinite(), x.abs(), 0.0).unflatten(-1, (-1, 128)).amax(dim=-1)
    e = torch.full(most.shape, -100, dtype=torch.int64)
    for up in range(-100, 121):
        e = torch.where(most > 448.0 * 2.0 ** up, up + 1, e)
    return torch.ldexp(torch.ones_like(most), e)


def quantized(x, scale=None):
    """(values of the codes, scales) in 64 bits."""
    x = x.double()
    scale = block_scales(x) if scale is None else scale
    v = x / scale.repeat_interleave(128, dim=-1)
    return torch.where(x.isfinite(), e4m3(torch.where(x.isfinite(), v, 0.0)), float("nan")), scale


def rounded(x):
    v, s = quantized(x)
    return v * s.repeat_interleave(128, dim=-1)


def weights(n, k, seed, lead=()):
    """e4m3 codes [.., n, k] and block scales on the CPU, and the weights in 64 bits."""
    g = torch.Generator().manual_seed(seed)
    codes = (torch.randn(lead + (n, k), generator=g) * 40).clamp_(-448, 448).to(F8)
    s = (torch.rand(lead + ((n + 127) // 128, k // 128), generator=g) + 0.5) * (k ** -0.5 / 40)
    s = s * torch.where(torch.rand(s.shape, generator=g) < 0.2, -1.0, 1.0)                   # scales may be negative
    w = codes.double() * s.double().repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)
    return codes, s, w


def product_error(x, w):
    """How far the sums x . w^T of the kernels may be off, [T, N].  The matrix cores add the products of eight consecutive k with 13 bits below the largest of them, cut off towards
    zero: at most 7 2^-13 of the largest, eight k at a time.  For weights and activations of random signs these are independent and of either sign, so the sum is
    within 6 sqrt(sum of their squares) (2 exp(-18) of not being so; a bounded variable's standard deviation is below its bound, here 0.1 of it).  Then the fp32 sums: two roundings
    of 2^-24 a window of 128 and two of the scales, each of at most the sum of magnitudes so far, 8 roundings of all of it."""
    t, k = x.shape
    biggest = torch.zeros(t, w.shape[0], dtype=torch.float64)
    total = torch.zeros_like(biggest)
    for i in range(0, k, 8):
        p = (x[:, None, i:i + 8] * w[None, :, i:i + 8]).abs()
        biggest += p.amax(dim=-1) ** 2
        total += p.sum(dim=-1)
    return 6 * 7 * 2.0 ** -13 * biggest.sqrt() + (8 + k / 256) * 2.0 ** -24 * total


def assert_within(got, want, error, dtype, what=""):
    """`error` of the sums and half a step of the result's type."""
    got = got.detach().cpu().double()
    tol = error * (1 + HALF[dtype]) + HALF[dtype] * want.abs() * 1.0001 + (2.0 ** -25 if dtype == torch.float16 else 1e-38)
    off = (got - want).abs()
    worst = (off - tol).max().item() if off.numel() else 0.0
    assert worst <= 0, "%s: off by %g more than allowed (largest error %g)" % (what, worst, off.max().item())


def layer(E, H, I, seed):
    c1, s1, w1 = weights(2 * I, H, seed, (E,))
    c2, s2, w2 = weights(H, I, seed + 1, (E,))
    return (c1, s1), (c2, s2), w1, w2


def experts(x, w1, w2, ids, wts, place=None):
    """(y, how far the kernels may be from it) [T, H] in 64 bits.  `place`: the expert map.  The intermediate h may be off by what the two sums are; a code of it then moves to a
    neighbour where a border lies that near, and the scale with its block's maximum: each element counts with the farthest value that h - error .. h + error can have."""
    T, H = x.shape
    I = w2.shape[2]
    xq = rounded(x)
    y, error = torch.zeros(T, H, dtype=torch.float64), torch.zeros(T, H, dtype=torch.float64)
    for t in range(T):
        for j in range(ids.shape[1]):
            e = int(ids[t, j])
            if place is not None:
                e = int(place[e]) if 0 <= e < place.numel() else -1
            if not 0 <= e < w1.shape[0]:
                continue
            row = xq[t:t + 1]
            both, off = row @ w1[e].t(), product_error(row, w1[e])
            g, u, og, ou = both[:, :I], both[:, I:], off[:, :I], off[:, I:]
            sig = torch.sigmoid(g)
            h = g * sig * u
            oh = 1.1 * u.abs() * og + (g * sig).abs() * ou + 1.1 * og * ou + 8 * 2.0 ** -24 * (1 + g.abs()) * h.abs()
            q = rounded(h)
            scales = [block_scales(v) for v in (h.abs() + oh, (h.abs() - oh).clamp(min=0))]
            far = torch.zeros_like(h)
            for s in scales:
                for v in (h - oh, h, h + oh):
                    wide = s.repeat_interleave(128, dim=-1)
                    far = torch.maximum(far, (e4m3((v / wide).clamp(-448, 448)) * wide - q).abs())
            wt = abs(float(wts[t, j]))
            y[t] += float(wts[t, j]) * (q @ w2[e].t())[0]
            error[t] += wt * (product_error(q, w2[e]) + far @ w2[e].abs().t())[0]
    return y, error
