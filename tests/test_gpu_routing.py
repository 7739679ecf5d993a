"""GPU: `moe_routing` and its gradient against the formulas in 64 bits on the CPU."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32
HALF = {HF: 2.0 ** -11, BF: 2.0 ** -8, F32: 2.0 ** -24}


def logits_of(T, E, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((T, E), generator=g) * spread + torch.randn(E, generator=g)).to(dtype)


def counted(logits):
    x = logits.double()
    return torch.where(x.isnan(), -math.inf, x).clamp(max=float(torch.finfo(torch.float32).max))


def picks(x, K, sigmoid, G, kept, bias):
    """ids by the definition, in 64 bits: -1 where no expert is left."""
    T, E = x.shape
    rank = x.clone()
    if bias is not None:
        top = x.max(dim=-1, keepdim=True)[0]
        score = torch.sigmoid(x) if sigmoid else torch.exp(x - torch.where(top.isinf(), 0.0, top))
        if not sigmoid:
            score = score / score.sum(dim=-1, keepdim=True)
        b = bias.double()
        rank = torch.where((x == -math.inf) | b.isnan(), -math.inf, score + b)
    ids = torch.full((T, K), -1, dtype=torch.int32)
    for t in range(T):
        r = rank[t].clone()
        if G > 1:
            each = r.view(G, -1)
            two = torch.sort(each, dim=-1, descending=True)[0]
            best = two[:, 0]
            if bias is not None and two.shape[1] > 1:
                best = torch.where(two[:, 1] == -math.inf, best, best + two[:, 1])
            order = sorted(range(G), key=lambda q: (-best[q].item(), q))
            for q in order[kept:]:
                r[q * (E // G):(q + 1) * (E // G)] = -math.inf
        for k in range(K):
            i = int(torch.argmax(r))                                # of equal ones the first below
            i = int((r == r[i]).nonzero()[0])
            if r[i] == -math.inf:
                break
            ids[t, k] = i
            r[i] = -math.inf
    return ids


def weights_of(x, ids, sigmoid, renorm, scaling):
    """Weights of given picks, in 64 bits, written so that torch can differentiate it."""
    here = ids >= 0
    at = ids.long().clamp(min=0)
    top = x.detach().max(dim=-1, keepdim=True)[0]
    top = torch.where(top.isinf(), 0.0, top)
    if sigmoid:
        log = torch.nn.functional.logsigmoid(x.gather(1, at))
    else:
        log = x.gather(1, at) if renorm else (x - top).gather(1, at) - torch.exp(x - top).sum(dim=-1, keepdim=True).clamp(min=1e-300).log()
    log = torch.where(here, log, -math.inf)
    if renorm:
        m = log.detach().max(dim=-1, keepdim=True)[0]
        s = torch.where(here, torch.exp(log - torch.where(m.isinf(), 0.0, m)), 0.0)
        return scaling * s / s.sum(dim=-1, keepdim=True).clamp(min=1e-300)
    return scaling * torch.where(here, torch.exp(log), 0.0)


def check(mlk, logits, K, sigmoid=False, renorm=True, G=1, kept=1, bias=None, scaling=1.0, mask=None, up=None):
    """ids equal.  Weights: exponentials and logistic functions good to 4 roundings, a sum of up to 512 of them to 10 (its tree's depth), a division and two products: 24
    roundings of 2^-24, and one to the type.  The gradient is s r (g - sum g s) or of that kind: 32 roundings of s (|g| + sum |g| s)."""
    T, E = logits.shape
    leaf = logits.cuda().requires_grad_(True)
    dev = [None if t is None else t.cuda() for t in (bias, mask)]
    ids, w = mlk.moe_routing(leaf, K, "sigmoid" if sigmoid else "softmax", renorm, G, kept, dev[0], scaling, dev[1])
    assert ids.dtype == torch.int32 and tuple(ids.shape) == (T, K) and w.dtype == logits.dtype and tuple(w.shape) == (T, K)
    x = counted(logits)
    if mask is not None:
        x[~mask] = 0.0
    want = picks(x, K, sigmoid, G, kept, bias)
    if mask is not None:
        want[~mask] = -1
    assert torch.equal(ids.cpu(), want)
    assert not ids.requires_grad
    x.requires_grad_(True)
    ww = weights_of(x, want, sigmoid, renorm, scaling)
    tiny = 2.0 ** -25 if logits.dtype == HF else 1e-38
    tol = (HALF[logits.dtype] * 1.001 + 24 * 2.0 ** -24) * ww.abs() + tiny
    off = (w.detach().cpu().double() - ww.detach()).abs()
    assert (off <= tol.detach()).all(), (off - tol).max().item()
    if up is None:
        up = torch.randn((T, K), generator=torch.Generator().manual_seed(T)).to(logits.dtype)
    grad, = torch.autograd.grad(w, leaf, grad_outputs=up.cuda())
    d, = torch.autograd.grad((ww * up.double()).sum(), x)
    d = torch.where(d.isnan(), 0.0, d)                       # of logits of -inf
    a = (up.double().abs() * abs(scaling)).masked_fill(want < 0, 0.0)
    share = ww.detach().abs() / abs(scaling)
    size = torch.zeros_like(d).scatter_add_(1, want.long().clamp(min=0), share * (a + (a * share).sum(dim=-1, keepdim=True)))
    if not sigmoid and not renorm:
        size = size + torch.softmax(x.detach(), dim=-1).nan_to_num() * (a * share).sum(dim=-1, keepdim=True)
    off = (grad.cpu().double() - d).abs()
    tol = HALF[logits.dtype] * 1.001 * d.abs() + 32 * 2.0 ** -24 * size + tiny
    assert grad.dtype == logits.dtype and (off <= tol).all(), (off - tol).max().item()
    with torch.no_grad():
        again = mlk.moe_routing(leaf, K, "sigmoid" if sigmoid else "softmax", renorm, G, kept, dev[0], scaling, dev[1])
    assert torch.equal(again[0], ids) and torch.equal(again[1], w) and not again[1].requires_grad
    return ids, w, grad


SIZES = [(1, 1, 1), (1, 8, 2), (3, 2, 2), (7, 64, 6), (33, 17, 17), (64, 65, 5), (100, 256, 8), (31, 257, 9), (16, 512, 32), (1025, 8, 2), (1030, 60, 4), (1027, 129, 8), (1031, 256, 20),
         (1026, 300, 3), (1029, 512, 10),
         (4100, 130, 5), (4097, 257, 3)]


@pytest.mark.parametrize("renorm", [True, False])
@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("T,E,K", SIZES)
def test_picks_weights_and_gradient(mlk, T, E, K, dtype, sigmoid, renorm):
    check(mlk, logits_of(T, E, dtype, T + E), K, sigmoid, renorm, scaling=1.0 if renorm else 2.5)


@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("T,E,K,G,kept", [(1, 256, 8, 8, 4), (50, 256, 8, 8, 4), (9, 24, 4, 3, 2), (33, 160, 6, 8, 3), (12, 16, 3, 16, 5), (20, 512, 32, 64, 8), (1100, 256, 8, 8, 4),
                                          (1030, 160, 6, 20, 3), (1027, 512, 8, 32, 16), (4100, 256, 8, 8, 4), (4101, 512, 8, 32, 16),
                                          (4098, 120, 7, 40, 9), (4103, 66, 4, 11, 5)])
def test_bias_groups_and_masks(mlk, T, E, K, G, kept, dtype, sigmoid):
    g = torch.Generator().manual_seed(E)
    bias = torch.randn(E, generator=g) * 0.2
    mask = torch.rand(T, generator=g) < 0.7
    x = logits_of(T, E, dtype, T)
    check(mlk, x, K, sigmoid, True, G, kept, bias, 2.5, mask)
    check(mlk, x, K, sigmoid, False, G, kept, None, 1.0, mask)
    check(mlk, x, K, sigmoid, True, 1, 1, bias)
    poisoned = x.clone()
    poisoned[~mask] = float("nan")
    check(mlk, poisoned, K, sigmoid, True, G, kept, bias, 1.0, mask)


@pytest.mark.parametrize("T", [6, 1030])
@pytest.mark.parametrize("sigmoid", [True, False])
@pytest.mark.parametrize("renorm", [True, False])
def test_infinities_nan_and_ties(mlk, T, sigmoid, renorm):
    E, K = 40, 5
    x = logits_of(T, E, F32, 3)
    x[0] = -math.inf                                         # nothing is left
    x[1, :38] = -math.inf                                    # less than is picked
    x[2, ::2] = float("nan")
    x[3] = 1.25                                              # ties everywhere
    x[4, 7], x[4, 9] = torch.finfo(F32).max, torch.finfo(F32).min           # the type's ends
    x[5] = torch.where(torch.arange(E) % 3 == 0, 0.0, -0.0)  # equal zeros
    check(mlk, x, K, sigmoid, renorm)
    bias = torch.zeros(E)
    bias[4], bias[5], bias[6] = -math.inf, float("nan"), 1e30
    check(mlk, x, K, sigmoid, renorm, 1, 1, bias)
    check(mlk, x, K, sigmoid, renorm, 8, 3, bias)
    x[4, 7] = math.inf                                       # the largest finite number
    check(mlk, x, K, sigmoid, renorm, 8, 3)
    ids, w = mlk.moe_routing(torch.full((3, 8), -math.inf, device="cuda"), 2)
    assert (ids == -1).all() and (w == 0).all()


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("level", [-300.0, -95.0, -20.0, 15.0, 80.0])
def test_scores_far_out(mlk, level, dtype):
    """Renormalised weights keep their bits where all scores vanish or all are 1."""
    x = (logits_of(64, 32, F32, 1) + level).to(dtype)
    check(mlk, x, 4, True, True)
    check(mlk, x, 4, False, True)


def test_gradient_against_differences(mlk):
    x = logits_of(4, 12, F32, 9).double()
    up = torch.randn(4, 3, generator=torch.Generator().manual_seed(2))
    for sigmoid in (False, True):
        for renorm in (False, True):
            leaf = x.float().cuda().requires_grad_(True)
            ids, w = mlk.moe_routing(leaf, 3, "sigmoid" if sigmoid else "softmax", renorm)
            grad, = torch.autograd.grad(w, leaf, grad_outputs=up.cuda())
            step = 1e-5                                      # differences in 64 bits: off by step^2 and 1e-16 / step, far below fp32's 1e-6
            for t in range(4):
                for e in range(12):
                    hi, lo = x.clone(), x.clone()
                    hi[t, e] += step
                    lo[t, e] -= step
                    d = ((weights_of(hi, ids.cpu(), sigmoid, renorm, 1.0) - weights_of(lo, ids.cpu(), sigmoid, renorm, 1.0)) * up.double()).sum() / (2 * step)
                    assert abs(grad[t, e].item() - d.item()) <= 4e-6


def test_neighbours_in_64_bits(mlk):
    """Scores + bias that fp32 cannot tell apart are ranked by their 64 bits: sigmoids of logits one fp32 step apart near 4 differ by 1e-8 and less."""
    base = torch.tensor(4.0)
    steps = [base]
    for _ in range(31):
        steps.append(torch.nextafter(steps[-1], torch.tensor(9.0)))
    x = torch.stack(steps)[torch.randperm(32, generator=torch.Generator().manual_seed(1))].expand(5, 32).contiguous()
    check(mlk, x, 32, True, True, 1, 1, torch.zeros(32))
    check(mlk, x.repeat(300, 1), 8, True, True, 1, 1, torch.full((32,), 1.0))


def test_calls(mlk):
    x = logits_of(70, 64, BF, 1).cuda()
    flat = torch.empty(70 * 64 + 1, dtype=BF, device="cuda")
    flat[1:] = x.flatten()
    off = flat[1:].view(70, 64)                              # off 8 bytes
    a, b = mlk.moe_routing(x, 6), mlk.moe_routing(off, 6)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    empty = mlk.moe_routing(x[:0].detach().requires_grad_(True), 6)
    assert empty[0].shape == (0, 6)
    empty[1].sum().backward()
    leaf = x.clone().requires_grad_(True)
    ids, w = mlk.moe_routing(leaf, 6)
    w.sum().backward()                                       # an expanded gradient
    first = leaf.grad.clone()
    g, = torch.autograd.grad(mlk.moe_routing(leaf, 6)[1], leaf, grad_outputs=torch.ones((6, 70), dtype=BF, device="cuda").t())
    assert torch.equal(first, g)
    ids, w = mlk.moe_routing(leaf, 6)
    grad, = torch.autograd.grad(w.float().square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        grad.float().sum().backward()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level(), pytest.raises(RuntimeError, match="forward-mode"):
        mlk.moe_routing(fwd.make_dual(x.float(), torch.ones_like(x).float()), 6)
    with pytest.raises(RuntimeError, match="gating_bias has no gradient"):
        mlk.moe_routing(x, 6, gating_bias=torch.zeros(64, device="cuda", requires_grad=True))


@pytest.mark.parametrize("T", [20, 2000])
def test_graph_replays_both_ways(mlk, T):
    leaf = logits_of(T, 256, F32, 1).cuda().requires_grad_(True)
    bias = torch.zeros(256, device="cuda")
    up = torch.randn(T, 8, device="cuda")

    def step():
        ids, w = mlk.moe_routing(leaf, 8, "sigmoid", True, 8, 4, bias, 2.5)
        return ids, w, torch.autograd.grad(w, leaf, grad_outputs=up)[0]

    def plain():
        return [t.detach().clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        plain()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    out = [t.detach() for t in out]
    for i in range(4):
        with torch.no_grad():
            leaf.copy_(logits_of(T, 256, F32, 30 + i))
            bias.copy_(torch.randn(256, generator=torch.Generator().manual_seed(i)) * 0.1)
        graph.replay()
        torch.cuda.synchronize()
        with torch.no_grad():
            ids, w = mlk.moe_routing(leaf, 8, "sigmoid", True, 8, 4, bias, 2.5)
        torch.cuda.synchronize()
        assert torch.equal(out[0], ids) and torch.equal(out[1], w)
        other = leaf.detach().clone().requires_grad_(True)
        _, w = mlk.moe_routing(other, 8, "sigmoid", True, 8, 4, bias, 2.5)
        grad, = torch.autograd.grad(w, other, grad_outputs=up)
        assert torch.equal(out[2], grad)


def test_with_the_balance_loss_and_the_experts(mlk):
    """A training step's router: the weights' gradient and the balance loss of the same picks reach the same logits."""
    T, E, K = 200, 16, 3
    leaf = logits_of(T, E, F32, 4).cuda().requires_grad_(True)
    up = torch.randn(T, K, device="cuda")
    ids, w = mlk.moe_routing(leaf, K)
    loss, counts = mlk.moe_balance_loss(leaf, ids, coef=0.01)
    both, = torch.autograd.grad((w * up).sum() + loss, leaf)
    other = leaf.detach().clone().requires_grad_(True)
    g1, = torch.autograd.grad((mlk.moe_routing(other, K)[1] * up).sum(), other)
    g2, = torch.autograd.grad(mlk.moe_balance_loss(other, ids, coef=0.01)[0], other)
    assert torch.allclose(both, g1 + g2, rtol=1e-6, atol=1e-9)
    assert torch.equal(counts, mlk.expert_counts(ids, E))
