"""Performance cases of the operators with 4-bit weights and of the router's balance statistics, each in its plain form (elementary torch
operations in 32 bits) and as a program calls the library.

  linear   `gemv_layoutA_w4` (one token) and `gemm_layoutA_w4`: y = x . W^T (+ bias), W[n, k] = s[n, k / G] (q[n, k] - z[n, k / G]) with codes q of
           4 bits, one 16-bit scale for every G weights of a row and, if `zeros`, one zero point of 4 bits beside it (8 otherwise)
  experts  `fused_experts_w4`: the two products of an expert layer over such weights, SiLU(gate) * up in between, weighted sum of a token's
           experts; the routing is an input.  `held` of the `experts` lie on this card, the others' pairs are dropped
  balance  `moe_balance_loss` and its gradient: per-expert counts, f = share of the routed pairs, P = sum of the router's probabilities,
           loss = coef mean over the sequences of E sum_e f_e P_e / n; masked tokens and rows behind the last sequence do not count
  counts   `expert_counts`: how often each expert was picked in a serving step

`rows` and `k` are those of the weight matrix, `tokens` the rows of the activations.
"""
import math

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}

# Weight shapes (rows, k) of the packaged launch-parameter tables and of the benchmark.
_SHAPES = [(4096, 4096), (11008, 4096), (4096, 11008), (12288, 4096), (22016, 4096), (32000, 4096), (8192, 8192), (28672, 4096),
           (4096, 14336), (28672, 8192), (8192, 14336), (4608, 3584), (37888, 3584), (3584, 18944), (4608, 7168), (7168, 2048),
           (512, 7168), (7168, 2304), (1280, 5120), (5120, 640), (13824, 5120), (5120, 13824), (10240, 8192), (27648, 5120)]
# Expert layers (experts, picks, hidden, intermediate): the benchmark's layer, a layer of the repository's tests, two of generic sizes.
_MOE = [(8, 2, 4096, 14336), (128, 8, 2048, 768), (16, 4, 4096, 2048), (64, 6, 2048, 1408)]
_MAX_FLOPS, _MAX_BYTES = 7.0e11, 7.4e8          # of the largest listed cases


def _linear(name, rows, k, tokens, dtype, group=128, zeros=False, bias=False):
    return {"name": name, "kind": "linear", "rows": rows, "k": k, "tokens": tokens, "dtype": dtype, "group": group, "zeros": zeros, "bias": bias}


def _experts(name, layer, tokens, dtype, group=128, zeros=False, held=None):
    e, picks, hidden, inter = layer
    return {"name": name, "kind": "experts", "experts": e, "held": e if held is None else held, "picks": picks, "hidden": hidden, "inter": inter,
            "tokens": tokens, "dtype": dtype, "group": group, "zeros": zeros}


def _balance(name, tokens, experts, picks, dtype, sigmoid=False, sequences=0, masked=False):
    return {"name": name, "kind": "balance", "tokens": tokens, "experts": experts, "picks": picks, "dtype": dtype, "sigmoid": sigmoid,
            "sequences": sequences, "masked": masked}


def _counts(name, tokens, experts, picks, masked):
    return {"name": name, "kind": "counts", "tokens": tokens, "experts": experts, "picks": picks, "masked": masked, "dtype": "bf16"}


def listed():
    return [
        # decode of one token through a small projection: launch latency counts
        _linear("gemv_bf16_512x7168", 512, 7168, 1, "bf16"),
        # decode of one token through a large feed-forward matrix, weights with zero points
        _linear("gemv_fp16_28672x8192_zeros", 28672, 8192, 1, "fp16", 128, True),
        # a decode batch of sixteen through a feed-forward matrix
        _linear("gemm_bf16_4096x14336_t16", 4096, 14336, 16, "bf16"),
        # an odd decode batch through a layer with small groups, zero points and a bias
        _linear("gemm_fp16_13824x5120_t37_g32", 13824, 5120, 37, "fp16", 32, True, True),
        # a long prompt
        _linear("gemm_bf16_27648x5120_t2048", 27648, 5120, 2048, "bf16"),
        # one token through an expert layer
        _experts("experts_bf16_8_t1", _MOE[0], 1, "bf16"),
        # a decode batch through many small experts, half of which another card holds
        _experts("experts_fp16_128_t50_held64", _MOE[1], 50, "fp16", 64, True, 64),
        # a prompt through a few large experts
        _experts("experts_bf16_8_t1000", _MOE[0], 1000, "bf16"),
        # the load of the experts in a serving step with padded rows
        _counts("counts_256experts_t64", 64, 256, 8, True),
        # the same over a long prompt
        _counts("counts_64experts_t30000", 30000, 64, 6, False),
        # a training step's balance loss over one batch
        _balance("balance_bf16_e64_t16384", 16384, 64, 6, "bf16"),
        # the loss of each sequence, fp32 router with normalised sigmoid scores, padded tokens, rows behind the last sequence
        _balance("balance_fp32_e256_t32749_seq9", 32749, 256, 8, "fp32", True, 9, True),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    while True:
        case = _draw(rng)
        if work(case)["bytes"] <= _MAX_BYTES:
            return case


def _draw(rng):
    kind = rng.choice(["linear", "linear", "linear", "experts", "experts", "balance", "balance", "counts"])
    group, zeros = rng.choice([32, 64, 128, 128]), rng.random() < 0.5
    if kind == "linear":
        rows, k = rng.choice(_SHAPES)
        if rng.random() < 0.5:
            rows, k = 16 * _log_int(rng, 8, 1792), 128 * _log_int(rng, 3, 64)
        tokens = 1 if rng.random() < 0.25 else _log_int(rng, 2, min(4096, _MAX_FLOPS / (2 * rows * k)))
        case = _linear("", rows, k, tokens, rng.choice(["bf16", "fp16"]), group, zeros, rng.random() < 0.3)
    elif kind == "experts":
        layer = rng.choice(_MOE)
        if rng.random() < 0.4:
            e = _log_int(rng, 4, 160)
            layer = (e, rng.randint(1, min(8, e)), 128 * _log_int(rng, 4, 32), 128 * _log_int(rng, 2, 16))
        e, picks, hidden, inter = layer
        tokens = _log_int(rng, 1, min(2048, _MAX_FLOPS / (6 * picks * hidden * inter)))
        held = None if rng.random() < 0.7 else rng.randint(1, e)
        case = _experts("", layer, tokens, rng.choice(["bf16", "fp16"]), group, zeros, held)
    elif kind == "balance":
        e = rng.choice([8, 16, 60, 64, 128, 160, 256])
        case = _balance("", _log_int(rng, 1, 32768), e, rng.randint(1, min(8, e)), rng.choice(["bf16", "fp16", "fp32"]), rng.random() < 0.5,
                        rng.choice([0, 0, 1, 3, 17]), rng.random() < 0.4)
    else:
        e = rng.choice([8, 16, 60, 64, 128, 160, 256])
        case = _counts("", _log_int(rng, 1, 32768), e, rng.randint(1, min(8, e)), rng.random() < 0.4)
    case.pop("name")
    return case


# ------------------------------------------------------------------------------------------------------------ inputs
def _codes(gen, rows, k):
    """Codes of normal weights, two in a byte: element 2 i in the low half."""
    q = (torch.randn((rows, k), generator=gen, device="cuda") * 2.6 + 8).round_().clamp_(0, 15).to(torch.uint8)
    return q[:, 0::2] | (q[:, 1::2] << 4)


def _weights(gen, rows, k, case):
    dtype, group = _DTYPE[case["dtype"]], case["group"]
    codes = _codes(gen, rows, k)
    scales = ((torch.rand((rows, k // group), generator=gen, device="cuda") + 0.5) * (k ** -0.5 / 2.6)).to(dtype)
    zeros = torch.randint(5, 12, (rows, k // group), generator=gen, device="cuda", dtype=torch.uint8) if case["zeros"] else None
    return codes, scales, zeros


def _expert_weights(gen, rows, k, case):
    made = [_weights(gen, rows, k, case) for _ in range(case["held"])]
    return tuple(None if part[0] is None else torch.stack(part) for part in zip(*made))


def _picks(gen, tokens, experts, picks):
    """Router logits, some experts more popular than others, and the experts with the largest ones, lowest index first."""
    logits = torch.randn((tokens, experts), generator=gen, device="cuda") + 0.5 * torch.randn(experts, generator=gen, device="cuda")
    return logits, torch.sort(logits, dim=-1, descending=True, stable=True)[1][:, :picks].to(torch.int32).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, tokens, dtype = case["kind"], case["tokens"], _DTYPE[case["dtype"]]
    state = {"kind": kind, "case": case}
    if kind == "linear":
        weights = _weights(gen, case["rows"], case["k"], case)
        state["x"] = torch.randn((tokens, case["k"]), generator=gen, device="cuda").to(dtype)
        state["bias"] = torch.randn((1, case["rows"]), generator=gen, device="cuda").to(dtype) if case["bias"] else None
        state["w"] = weights
    elif kind == "experts":
        e, held, hidden, inter = case["experts"], case["held"], case["hidden"], case["inter"]
        w1, w2 = _expert_weights(gen, 2 * inter, hidden, case), _expert_weights(gen, hidden, inter, case)
        state["x"] = torch.randn((tokens, hidden), generator=gen, device="cuda").to(dtype)
        logits, state["ids"] = _picks(gen, tokens, e, case["picks"])
        p = torch.gather(torch.exp(logits), 1, state["ids"].long())
        state["weights"] = (p / p.sum(dim=-1, keepdim=True)).to(dtype)
        state["map"] = None
        if held < e:
            state["map"] = torch.full((e,), -1, dtype=torch.int32, device="cuda")
            here = torch.randperm(e, generator=gen, device="cuda")[:held].sort()[0]
            state["map"][here] = torch.arange(held, dtype=torch.int32, device="cuda")
        state["w1"], state["w2"] = w1, w2
    else:
        logits, state["ids"] = _picks(gen, tokens, case["experts"], case["picks"])
        state["mask"] = torch.rand(tokens, generator=gen, device="cuda") < 0.8 if case["masked"] else None
        if kind == "balance":
            state["logits"] = logits.to(dtype).requires_grad_(True)
            # fp16 gradients need a scaled loss, as a training program in fp16 has
            state["up"] = torch.tensor(65536.0 if case["dtype"] == "fp16" else 1.0, device="cuda")
            state["cu"] = None
            if case["sequences"]:
                # lengths at random, the second of several empty, some rows behind the last sequence
                cuts = torch.randint(0, max(1, tokens - tokens // 50) + 1, (case["sequences"] + 1,), generator=gen, device="cuda").sort()[0]
                cuts[0] = 0
                cuts[-1] = tokens - tokens // 50
                if case["sequences"] > 2:
                    cuts[2] = cuts[1]
                state["cu"] = cuts.to(torch.int32)
    if own:
        # what a program keeps of its weights: the library's layout, packed once at load time, in place of the checkpoint's rows
        import muxi_layout_kernels as mlk
        for name in ("w", "w1", "w2"):
            if name in state:
                state[name] = mlk.pack_layout_a_w4(*state[name])
    return state


# -------------------------------------------------------------------------------------------------------- plain forms
def _dequantised(codes, scales, zeros):
    """[.., rows, k / 2] codes, [.., rows, k / G] scales and zero points -> fp32 weights [.., rows, k]."""
    q = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2).float()
    q = q.unflatten(-1, (scales.shape[-1], -1))
    z = 8.0 if zeros is None else zeros.float().unsqueeze(-1)
    return ((q - z) * scales.float().unsqueeze(-1)).flatten(-2)


def _plain_linear(state):
    y = state["x"].float() @ _dequantised(*state["w"]).t()
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(state["x"].dtype)


def _plain_experts(state):
    x, ids, held = state["x"].float(), state["ids"].long(), state["case"]["held"]
    if state["map"] is not None:
        ids = state["map"].long()[ids]
    w1, w2 = state["w1"], state["w2"]
    share = state["weights"].float().unsqueeze(-1) * (ids.unsqueeze(-1) == torch.arange(held, device=x.device))
    share = share.sum(dim=1)                                                # [tokens, held]
    if x.shape[0] == 1 and ids.shape[1] < held:                             # one token: only its experts' weights are read
        ids = ids.clamp(min=0)[0]
        w1, w2 = (tuple(None if p is None else p[ids] for p in w) for w in (w1, w2))
        share = share[:, ids]
    w1, w2 = _dequantised(*w1), _dequantised(*w2)                           # [e, 2 I, H], [e, H, I]
    e, hidden, inter = w2.shape
    gate, up = (x @ w1.reshape(e * 2 * inter, hidden).t()).view(-1, e, 2, inter).unbind(2)
    h = gate / (1 + torch.exp(-gate)) * up * share.unsqueeze(-1)
    return (h.reshape(-1, e * inter) @ w2.transpose(1, 2).reshape(e * inter, hidden)).to(state["x"].dtype)


def _plain_counts(ids, mask, experts):
    hit = ids.unsqueeze(-1) == torch.arange(experts, device=ids.device)
    if mask is not None:
        hit = hit & mask.view(-1, 1, 1)
    return hit.sum(dim=(0, 1)).to(torch.int32)


def _plain_balance(state):
    logits, ids, cu = state["logits"].detach().float(), state["ids"], state["cu"]
    tokens, experts = logits.shape
    picks = ids.shape[1]
    place = torch.arange(tokens, device=logits.device)
    if cu is None:
        inside = torch.ones((1, tokens), dtype=torch.bool, device=logits.device)
    else:
        inside = (place >= cu[:-1].unsqueeze(1)) & (place < cu[1:].unsqueeze(1))           # [sequences, tokens]
    if state["mask"] is not None:
        inside = inside & state["mask"]
    inside = inside.float()
    if state["case"]["sigmoid"]:
        score = 1 / (1 + torch.exp(-logits))
    else:
        score = torch.exp(logits - logits.max(dim=-1, keepdim=True)[0])
    p = score / score.sum(dim=-1, keepdim=True)
    hits = (ids.unsqueeze(-1) == torch.arange(experts, device=ids.device)).sum(dim=1).float()      # [tokens, experts]
    n = inside.sum(dim=1, keepdim=True)
    c = inside @ hits
    g = c * (experts / picks) / torch.where(n > 0, n * n, 1.0) / torch.clamp((n > 0).sum(), min=1)
    loss = (g * (inside @ p)).sum()
    gt = inside.t() @ g                                                                            # each token's row of g, 0 where it counts nowhere
    dp = p * (gt - (p * gt).sum(dim=-1, keepdim=True))
    if state["case"]["sigmoid"]:
        dp = dp * (1 - score)
    return loss, c.sum(dim=0).to(torch.int32), (dp * state["up"]).to(state["logits"].dtype)


def run(state):
    kind = state["kind"]
    if own:
        import muxi_layout_kernels as mlk
        if kind == "linear":
            w, scale, zero = state["w"]
            product = mlk.gemv_layoutA_w4 if state["x"].shape[0] == 1 else mlk.gemm_layoutA_w4
            return product(w, scale, state["x"], zero, bias=state["bias"])
        if kind == "experts":
            (w1, s1, z1), (w2, s2, z2) = state["w1"], state["w2"]
            return mlk.fused_experts_w4(state["x"], w1, w2, state["ids"], state["weights"], s1, s2, z1, z2, experts_map=state["map"])
        if kind == "counts":
            return mlk.expert_counts(state["ids"], state["case"]["experts"], token_mask=state["mask"])
        loss, counts = mlk.moe_balance_loss(state["logits"], state["ids"], "sigmoid" if state["case"]["sigmoid"] else "softmax",
                                            token_mask=state["mask"], cu_seqlens=state["cu"])
        grad, = torch.autograd.grad(loss, state["logits"], grad_outputs=state["up"])
        return loss.detach(), counts, grad
    if kind == "linear":
        return _plain_linear(state)
    if kind == "experts":
        return _plain_experts(state)
    if kind == "counts":
        return _plain_counts(state["ids"], state["mask"], state["case"]["experts"])
    return _plain_balance(state)


# --------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    """Weights, scales and activations read once, outputs written once; two operations per weight and token.  Of an expert layer, the experts
    that even routing would be expected to reach and the pairs that stay on this card.  Of the balance loss, the logits read and their gradient written
    (some ten operations each), the picks and the mask read."""
    tokens, size = case["tokens"], 4 if case["dtype"] == "fp32" else 2

    def matrix(rows, k):
        return rows * k // 2 + rows * (k // case["group"]) * (3 if case["zeros"] else 2)

    if case["kind"] == "linear":
        rows, k = case["rows"], case["k"]
        return {"bytes": matrix(rows, k) + 2 * tokens * (k + rows) + (2 * rows if case["bias"] else 0), "flops": 2 * tokens * rows * k}
    picks, e = case["picks"], case["experts"]
    if case["kind"] == "experts":
        hidden, inter = case["hidden"], case["inter"]
        reached = case["held"] * (1 - (1 - picks / e) ** tokens)
        pairs = tokens * picks * case["held"] / e
        return {"bytes": reached * (matrix(2 * inter, hidden) + matrix(hidden, inter)) + 4 * tokens * hidden + 6 * tokens * picks,
                "flops": 6 * pairs * hidden * inter}
    read = 4 * tokens * picks + (tokens if case["masked"] else 0)
    if case["kind"] == "counts":
        return {"bytes": read + 4 * e, "flops": tokens * picks}
    return {"bytes": read + 2 * size * tokens * e + 4 * e, "flops": 10 * tokens * e}


# ------------------------------------------------------------------------------------------------- the definition in 64 bits
def _inputs(case, seed):
    """The inputs of `prepare` as a plain program has them."""
    global own
    was, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = was


def _table64(codes, scales, zeros):
    """Every weight from the table of the sixteen values of its group: value[n, group, code]."""
    rows, half = codes.shape
    zero = torch.full(scales.shape, 8, dtype=torch.float64, device=codes.device) if zeros is None else zeros.double()
    value = scales.double().unsqueeze(-1) * (torch.arange(16, dtype=torch.float64, device=codes.device) - zero.unsqueeze(-1))
    code = torch.empty((rows, 2 * half), dtype=torch.int64, device=codes.device)
    code[:, 0::2] = codes.long() % 16
    code[:, 1::2] = codes.long() // 16
    return torch.gather(value, 2, code.view(rows, scales.shape[1], -1)).view(rows, 2 * half)


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "counts":
        return None
    if kind == "linear":
        out = torch.nn.functional.linear(s["x"].double(), _table64(*s["w"]))
        return out if s["bias"] is None else out + s["bias"].double()
    if kind == "experts":
        x, out = s["x"].double(), torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
        for e in range(case["held"]):
            hit = (s["ids"] if s["map"] is None else s["map"][s["ids"].long()]) == e
            token, pick = hit.nonzero(as_tuple=True)
            if token.numel():
                part = lambda w: tuple(None if p is None else p[e] for p in w)       # noqa: E731
                both = torch.nn.functional.linear(x[token], _table64(*part(s["w1"])))
                h = torch.nn.functional.silu(both[:, :case["inter"]]) * both[:, case["inter"]:]
                out.index_add_(0, token, torch.nn.functional.linear(h, _table64(*part(s["w2"]))) * s["weights"][token, pick].double().unsqueeze(1))
        return out
    # loss of each sequence from its own rows; the gradient from torch's differentiation of it
    leaf = s["logits"].detach().double().requires_grad_(True)
    bounds = [0, case["tokens"]] if s["cu"] is None else s["cu"].tolist()
    terms = []
    for a, b in zip(bounds[:-1], bounds[1:]):
        keep = torch.arange(a, b, device="cuda") if s["mask"] is None else a + s["mask"][a:b].nonzero().flatten()
        if keep.numel():
            f = torch.bincount(s["ids"][keep].flatten().long(), minlength=case["experts"]).double() / (keep.numel() * case["picks"])
            rows = leaf[keep]
            p = torch.sigmoid(rows) if case["sigmoid"] else torch.softmax(rows, dim=-1)
            terms.append(case["experts"] * (f * (p / p.sum(dim=-1, keepdim=True)).mean(dim=0)).sum())
    if not terms:
        return torch.zeros((), dtype=torch.float64, device="cuda"), None, torch.zeros_like(leaf).detach()
    loss = torch.stack(terms).mean()
    grad, = torch.autograd.grad(loss, leaf)
    return loss.detach(), None, grad * s["up"].double()
