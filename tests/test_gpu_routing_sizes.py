"""GPU: `moe_routing` with more tokens than one launch has threads for."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_more_tokens_than_a_launch_takes(mlk):
    """2^28 tokens and 13 more of two experts, both ways: 16 threads a token are more than 2^32.  The rows around each 2^27 and random others are checked against the definition."""
    T, E, K = (1 << 28) + 13, 2, 1
    g = torch.Generator(device="cuda").manual_seed(1)
    logits = torch.empty((T, E), dtype=torch.float16, device="cuda")
    for part in logits.split(1 << 26):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda", dtype=torch.float16))
    logits.requires_grad_(True)
    mask = torch.ones(T, dtype=torch.bool, device="cuda")
    mask[::3] = False
    ids, w = mlk.moe_routing(logits, K, "sigmoid", False, token_mask=mask)
    up = torch.ones((1, 1), dtype=torch.float16, device="cuda").expand(T, K)
    grad, = torch.autograd.grad(w, logits, grad_outputs=up)
    edges = torch.cat([torch.arange(c - 40, min(c + 40, T), device="cuda") for c in (40, 1 << 27, 1 << 28, T)])
    rows = torch.cat([edges[edges < T], torch.randint(0, T, (20000,), generator=g, device="cuda")])
    x, here = logits.detach()[rows].double(), mask[rows].unsqueeze(1)
    best = torch.where(x[:, :1] >= x[:, 1:], 0, 1)
    assert torch.equal(ids[rows], torch.where(here, best, -1).int())
    s = torch.sigmoid(x.gather(1, best))
    half = 2.0 ** -11 * 1.001
    assert ((w.detach()[rows].double() - s * here).abs() <= half * s + 2.0 ** -25).all()
    want = torch.zeros_like(x).scatter(1, best, s * (1 - s) * here)
    assert ((grad[rows].double() - want).abs() <= half * want + 2.0 ** -25 + 8 * 2.0 ** -24 * want).all()
