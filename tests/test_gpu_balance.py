"""GPU: `moe_balance_loss`, its gradient and `expert_counts` against the formulas in 64 bits on the CPU."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def case(T, E, K, dtype, seed, spread=1.0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn((T, E), generator=g) * spread + torch.randn(E, generator=g)).to(dtype)
    ids = torch.stack([torch.randperm(E, generator=g)[:K] for _ in range(T)]).to(torch.int32) if T else torch.zeros((0, K), dtype=torch.int32)
    return logits, ids


def expected(logits, ids, sigmoid, coef, mask, cu):
    """loss, counts, gradient of the loss in 64 bits from the formulas; and p, g for the tolerances."""
    x = logits.double()
    T, E = x.shape
    K = ids.shape[1]
    if sigmoid:
        sig = torch.sigmoid(x)
        score = sig
    else:
        top = x.max(dim=-1, keepdim=True)[0]
        score = torch.exp(x - torch.where(torch.isinf(top), 0.0, top))
        sig = torch.zeros_like(x)
    total = score.sum(dim=-1, keepdim=True)
    p = torch.where(total > 0, score / total, 0.0)
    bounds = [0, T] if cu is None else cu.tolist()
    keep = torch.ones(T, dtype=torch.bool) if mask is None else mask
    counts, loss, g = torch.zeros(E, dtype=torch.int64), 0.0, torch.zeros(T, E, dtype=torch.float64)
    rows = [torch.arange(a, b)[keep[a:b]] for a, b in zip(bounds[:-1], bounds[1:])]
    rows = [r for r in rows if r.numel()]
    for r in rows:
        c = torch.bincount(ids[r].flatten().long().clamp(min=0), weights=((ids[r] >= 0) & (ids[r] < E)).flatten().double(), minlength=E)[:E]
        counts += c.long()
        share = coef / len(rows) * E / (K * r.numel() ** 2) * c
        loss += (share * p[r].sum(dim=0)).sum().item()
        g[r] = share
    grad = p * (1 - sig) * (g - (p * g).sum(dim=-1, keepdim=True))
    return loss, counts, torch.where(g.sum(dim=-1, keepdim=True) > 0, grad, 0.0), p, g


def check(mlk, logits, ids, sigmoid=False, coef=1.0, mask=None, cu=None, up=1.0):
    """Sums of at most 200 positive terms in a row and probabilities good to 16 roundings: 2e-5 of the loss.  The gradient is p (g - sum p g): 64 roundings of
    p max(g), and one to its type."""
    leaf = logits.cuda().requires_grad_(True)
    dev = [None if t is None else t.cuda() for t in (ids, mask, cu)]
    loss, counts = mlk.moe_balance_loss(leaf, dev[0], "sigmoid" if sigmoid else "softmax", coef, dev[1], dev[2])
    grad, = torch.autograd.grad(loss, leaf, grad_outputs=torch.tensor(up, device="cuda"))
    safe = logits if mask is None else torch.where(mask.unsqueeze(1), logits, torch.zeros_like(logits))
    want, c, d, p, g = expected(safe, ids, sigmoid, coef, mask, cu)
    assert loss.dtype == torch.float32 and loss.shape == () and counts.dtype == torch.int32
    assert abs(loss.item() - want) <= 2e-5 * abs(want)
    assert torch.equal(counts.cpu().long(), c)
    d = d * up
    tiny = 2.0 ** -25 if logits.dtype == torch.float16 else 1e-38
    tol = torch.finfo(logits.dtype).eps / 2 * d.abs() * 1.001 + 64 * 2.0 ** -24 * p * g.max(dim=-1, keepdim=True)[0] * abs(up) + tiny
    err = (grad.cpu().double() - d).abs()
    assert (err <= tol).all(), (err - tol).max().item()
    assert grad.dtype == logits.dtype
    return loss, counts, grad


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,E,K", [(1, 8, 2), (3, 1, 1), (31, 6, 3), (33, 17, 2), (64, 33, 8), (1000, 60, 4), (257, 64, 6), (555, 129, 5), (2049, 256, 8),
                                   (20000, 16, 2)])
def test_loss_counts_and_gradient(mlk, T, E, K, dtype, sigmoid):
    logits, ids = case(T, E, K, dtype, T + E)
    check(mlk, logits, ids, sigmoid, 0.01 if dtype == torch.float32 else 1.0, up=65536.0 if dtype == torch.float16 else 1.0)


@pytest.mark.parametrize("sigmoid", [False, True])
@pytest.mark.parametrize("cu", [[0, 700], [0, 0, 700, 700], [0, 1, 2, 3, 650], [5, 37, 37, 300, 301, 640], [0] * 70 + [300] * 5 + [699], [0, 0], [700, 700],
                                list(range(0, 700, 9)), [3]])
def test_sequences_and_masked_tokens(mlk, cu, sigmoid):
    T, E, K = 700, 40, 3
    logits, ids = case(T, E, K, torch.float32, len(cu))
    g = torch.Generator().manual_seed(5)
    cu = torch.tensor(cu, dtype=torch.int32)
    check(mlk, logits, ids, sigmoid, 1.0, None, cu)
    mask = torch.rand(T, generator=g) < 0.5
    mask[300:302] = False
    logits[~mask] = float("nan")                       # padding may hold anything
    _, _, grad = check(mlk, logits, ids, sigmoid, 1.0, mask, cu)
    outside = torch.ones(T, dtype=torch.bool)
    outside[int(cu[0]):int(cu[-1])] = False
    assert (grad.cpu()[outside | ~mask] == 0).all()
    nobody = torch.zeros(T, dtype=torch.bool)
    loss, counts, grad = check(mlk, logits, ids, sigmoid, 1.0, nobody, cu)
    assert loss.item() == 0 and (counts == 0).all() and (grad == 0).all()


@pytest.mark.parametrize("sigmoid", [False, True])
def test_extreme_logits_and_ids(mlk, sigmoid):
    T, E, K = 40, 24, 4
    logits, ids = case(T, E, K, torch.float32, 1)
    logits[3] = float("-inf")                          # no probability anywhere
    logits[4, 5:] = float("-inf")
    logits[5] = torch.finfo(torch.float32).min / 2 if not sigmoid else -60.0
    logits[6, 0] = 80.0
    ids[7] = torch.tensor([-1, E, 1 << 30, -(1 << 30)], dtype=torch.int32)
    ids[8] = 2                                         # one expert four times
    check(mlk, logits, ids, sigmoid)


def test_gradient_against_differences(mlk):
    T, E, K = 24, 10, 2
    for sigmoid in (False, True):
        logits, ids = case(T, E, K, torch.float32, 9)
        cu = torch.tensor([0, 7, 20], dtype=torch.int32)
        _, _, grad = check(mlk, logits, ids, sigmoid, 1.0, None, cu)
        for t, e in ((0, 0), (6, 3), (7, 9), (19, 4), (22, 1)):
            step = torch.zeros_like(logits, dtype=torch.float64)
            step[t, e] = 1e-4
            hi, lo = (expected(logits.double() + s, ids, sigmoid, 1.0, None, cu)[0] for s in (step, -step))
            assert abs((hi - lo) / 2e-4 - grad[t, e].item()) <= 1e-6


def test_empty_batch_and_no_sequence(mlk):
    logits = torch.zeros((0, 8), device="cuda", requires_grad=True)
    loss, counts = mlk.moe_balance_loss(logits, torch.zeros((0, 2), dtype=torch.int32, device="cuda"))
    loss.backward()
    assert loss.item() == 0 and (counts == 0).all() and logits.grad.shape == (0, 8)
    assert torch.equal(mlk.expert_counts(torch.zeros((0, 2), dtype=torch.int32, device="cuda"), 8), torch.zeros(8, dtype=torch.int32, device="cuda"))


def test_results_repeat_bit_for_bit_on_other_streams(mlk):
    logits, ids = case(5000, 100, 6, torch.bfloat16, 2)
    leaf, ids = logits.cuda().requires_grad_(True), ids.cuda()
    cu = torch.tensor([0, 100, 4000, 4990], dtype=torch.int32, device="cuda")

    def once():
        loss, counts = mlk.moe_balance_loss(leaf, ids, cu_seqlens=cu)
        return loss.detach(), counts, torch.autograd.grad(loss, leaf)[0]
    want = once()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(once())
    torch.cuda.synchronize()
    for out in got:
        assert all(torch.equal(a, b) for a, b in zip(out, want))


def test_unscaled_and_repeated_backward(mlk):
    logits, ids = case(100, 32, 2, torch.float32, 4)
    leaf = logits.cuda().requires_grad_(True)
    other = leaf * 2.0                                 # not a leaf
    loss, _ = mlk.moe_balance_loss(other, ids.cuda(), coef=0.5)
    (3.0 * loss).backward(retain_graph=True)
    first = leaf.grad.clone()
    (3.0 * loss).backward()
    assert torch.equal(leaf.grad, 2 * first)
    _, _, d, p, g = expected(logits.double() * 2, ids, False, 0.5, None, None)
    assert ((first.cpu().double() - 6 * d).abs() <= 6 * (65 * 2.0 ** -24 * p * g.max() + 2.0 ** -23 * d.abs())).all()


@pytest.mark.parametrize("T,E,K", [(1, 4, 1), (7, 256, 8), (64, 60, 6), (30000, 64, 6)])
def test_counts(mlk, T, E, K):
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(-2, E + 2, (T, K), generator=g, dtype=torch.int32)
    mask = torch.rand(T, generator=g) < 0.5
    for m in (None, mask):
        kept = (ids if m is None else ids[m]).flatten().long()
        want = torch.bincount(kept[(kept >= 0) & (kept < E)], minlength=E).int()
        got = mlk.expert_counts(ids.cuda(), E, token_mask=None if m is None else m.cuda())
        assert got.dtype == torch.int32 and torch.equal(got.cpu(), want)
        again = mlk.expert_counts(ids.cuda(), E, token_mask=None if m is None else m.cuda(), out=got)
        assert again is got and torch.equal(got.cpu(), 2 * want)


@pytest.mark.parametrize("sigmoid", [False, True])
def test_many_short_sequences(mlk, sigmoid):
    g = torch.Generator().manual_seed(8)
    T, E, K = 5000, 20, 2
    logits, ids = case(T, E, K, torch.float32, 3)
    cuts = torch.randint(0, T + 1, (1500,), generator=g).sort()[0].int()                     # some of them empty
    mask = torch.rand(T, generator=g) < 0.6
    check(mlk, logits, ids, sigmoid, 1.0, None, cuts)
    check(mlk, logits, ids, sigmoid, 1.0, mask, cuts)


def test_a_second_derivative_is_refused(mlk):
    logits, ids = case(50, 16, 2, torch.float32, 6)
    leaf = logits.cuda().requires_grad_(True)
    loss, counts = mlk.moe_balance_loss(leaf, ids.cuda())
    assert not counts.requires_grad
    plain, = torch.autograd.grad(loss, leaf, retain_graph=True)
    grad, = torch.autograd.grad(loss, leaf, create_graph=True)
    assert torch.equal(grad.detach(), plain)
    with pytest.raises(RuntimeError, match="cannot be differentiated again"):
        (grad.sum() + (leaf * leaf).sum()).backward()
    with torch.no_grad():
        quiet, _ = mlk.moe_balance_loss(leaf, ids.cuda())
    assert not quiet.requires_grad and torch.equal(quiet, loss.detach())


def test_forward_mode_is_refused(mlk):
    """A tangent would be dropped: of the logits, of the gradient that comes in.  A plain tensor in a dual level is as good as outside."""
    from torch.autograd import forward_ad
    logits, ids = case(40, 16, 2, torch.float32, 7)
    logits, ids = logits.cuda(), ids.cuda()
    want = mlk.moe_balance_loss(logits, ids)[0]
    leaf = logits.clone().requires_grad_(True)
    with forward_ad.dual_level():
        assert torch.equal(mlk.moe_balance_loss(logits, ids)[0], want)
        for x in (logits, leaf):
            dual = forward_ad.make_dual(x, torch.ones_like(x))
            with pytest.raises(RuntimeError, match="forward-mode"):
                mlk.moe_balance_loss(dual, ids)
            with torch.no_grad(), pytest.raises(RuntimeError, match="forward-mode"):
                mlk.moe_balance_loss(dual, ids)
        loss, _ = mlk.moe_balance_loss(leaf, ids)
        up = forward_ad.make_dual(torch.ones((), device="cuda"), torch.ones((), device="cuda"))
        with pytest.raises(RuntimeError, match="forward-mode"):
            torch.autograd.grad(loss, leaf, grad_outputs=up)
    with pytest.raises(RuntimeError):
        torch.func.jvp(lambda x: mlk.moe_balance_loss(x, ids)[0], (logits,), (torch.ones_like(logits),))
    with pytest.raises(RuntimeError):
        torch.func.grad(lambda x: mlk.moe_balance_loss(x, ids)[0])(logits)


def relative(mlk, logits, ids, E):
    """The largest error of the gradient's elements relative to their own size, where g - sum p g is not small against g (its own rounding counts there)."""
    leaf = logits.cuda().requires_grad_(True)
    loss, _ = mlk.moe_balance_loss(leaf, ids.cuda(), "sigmoid")
    grad, = torch.autograd.grad(loss, leaf)
    want, _, d, p, g = expected(logits, ids, True, 1.0, None, None)
    assert abs(loss.item() - want) <= 2e-5 * want
    clear = ((g - (p * g).sum(dim=-1, keepdim=True)).abs() > 0.1 * g.max()) & (d.abs() > 1e-30)
    assert clear.sum() > 100
    return ((grad.cpu().double() - d).abs() / d.abs())[clear].max().item()


def test_sigmoid_saturated_upwards(mlk):
    """1 - sigmoid of logits up to 15 keeps its bits: a gradient is a product of p, that and g - sum p g, each good to some ten roundings, of the last
    of which a tenth of g may remain: 200 * 2^-24."""
    T, E, K = 60, 16, 2
    logits, ids = case(T, E, K, torch.float32, 11)
    ids[:] = torch.tensor([3, 5], dtype=torch.int32)             # shares far apart
    assert relative(mlk, logits + 0.2 * torch.arange(T).unsqueeze(1), ids, E) <= 200 * 2.0 ** -24


def test_sigmoid_far_below_zero(mlk):
    """Sigmoids over their sum are a distribution however small they are: rows around -20 to -500, where fp32 has no such sigmoids; tolerance as above, and the logits' own
    rounding in x - max, which is exact."""
    T, E, K = 60, 16, 2
    logits, ids = case(T, E, K, torch.float32, 12)
    ids[:] = torch.tensor([3, 5], dtype=torch.int32)
    below = torch.cat((torch.linspace(-20, -110, 40), torch.linspace(-120, -500, 20))).unsqueeze(1)
    logits = logits + below
    assert relative(mlk, logits, ids, E) <= 200 * 2.0 ** -24
    logits[5:10, 8:] = float("-inf")                     # some experts out of the question
    logits[30:35, 8:] = float("-inf")
    logits[50:55, 8:] = float("-inf")
    assert relative(mlk, logits, ids, E) <= 200 * 2.0 ** -24
    logits[35] = torch.tensor([-100.0] * 15 + [3.0])     # one expert takes all
    check(mlk, logits, ids, True)
    for dtype in (torch.float16, torch.bfloat16):
        check(mlk, logits.to(dtype), ids, True, up=65536.0 if dtype == torch.float16 else 1.0)
    check(mlk, torch.full((7, 8), -95.0), torch.zeros((7, 2), dtype=torch.int32), True)
    check(mlk, torch.full((7, 256), -3.0e38), torch.zeros((7, 2), dtype=torch.int32))
