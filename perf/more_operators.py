"""Performance cases of the products in 8-bit floating point (e4m3) with a scale for each block of 128, of the expert layers over them and of
the router that trains, each in its plain form (elementary torch operations in 32 bits) and as a program calls the library.

  quantize  `quantize_fp8`: rows of activations to e4m3 codes and a power of two for every 128 of a row, the smallest (2^-100 at least) with
            max |x| <= 448 scale; an infinity or NaN becomes the NaN code and does not count in the maximum
  linear    `gemm_layoutA_fp8`: y = xq . W^T (+ bias), xq the activations as `quantize` leaves them, W[n, k] = s[n / 128, k / 128] q[n, k]
            with e4m3 codes q; activations go in as they are, the call quantises them
  experts   `fused_experts_fp8`: the two products of an expert layer over such weights; SiLU(gate) * up is quantised like activations in
            between; weighted sum of a token's experts; the routing is an input.  `held` of the `experts` lie on this card, the others'
            pairs are dropped
  routing   `moe_routing`: the `picks` experts of largest logit, or of largest score + bias, from the `kept` best of `groups` groups (their largest
            logit, or the sum of their two largest), lowest index first; weights are the scores (softmax or sigmoid), divided by the picks'
            sum if `renormalize`, times `scaling`; masked tokens get ids of -1 and weights of 0.  With `grad` also the gradient of the logits

`rows` and `k` are those of the weight matrix, `tokens` the rows of the activations.
"""
import math

import torch

own = False

_DTYPE = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_E4M3 = torch.float8_e4m3fn

# Weight shapes (rows, k) of the packaged launch-parameter tables and of the benchmark.
_SHAPES = [(4096, 4096), (11008, 4096), (4096, 11008), (12288, 4096), (22016, 4096), (32000, 4096), (8192, 8192), (28672, 4096),
           (4096, 14336), (28672, 8192), (8192, 14336), (4608, 3584), (37888, 3584), (3584, 18944), (4608, 7168), (7168, 2048),
           (512, 7168), (7168, 2304), (1280, 5120), (5120, 640), (13824, 5120), (5120, 13824), (10240, 8192), (27648, 5120)]
# Expert layers (experts, picks, hidden, intermediate): the benchmark's layer, a layer of the repository's tests, two of generic sizes.
_MOE = [(8, 2, 4096, 14336), (128, 8, 2048, 768), (16, 4, 4096, 2048), (64, 6, 2048, 1408)]
# Routers (experts, picks, groups, kept).
_ROUTERS = [(8, 2, 1, 1), (64, 6, 1, 1), (128, 8, 1, 1), (256, 8, 8, 4), (160, 6, 8, 3), (512, 10, 1, 1)]
_MAX_FLOPS, _MAX_BYTES = 5.4e11, 4.0e8          # of the largest listed cases
_MAX_PLAIN = 2.8e12                             # operations of the plain form of an expert layer, which takes every expert for every token


def _quantize(name, tokens, k, dtype):
    return {"name": name, "kind": "quantize", "tokens": tokens, "k": k, "dtype": dtype}


def _linear(name, rows, k, tokens, dtype, bias=False):
    return {"name": name, "kind": "linear", "rows": rows, "k": k, "tokens": tokens, "dtype": dtype, "bias": bias}


def _experts(name, layer, tokens, dtype, held=None):
    e, picks, hidden, inter = layer
    return {"name": name, "kind": "experts", "experts": e, "held": e if held is None else held, "picks": picks, "hidden": hidden, "inter": inter,
            "tokens": tokens, "dtype": dtype}


def _routing(name, tokens, router, dtype, sigmoid=False, bias=False, renormalize=True, masked=False, grad=True, scaling=1.0):
    e, picks, groups, kept = router
    return {"name": name, "kind": "routing", "tokens": tokens, "experts": e, "picks": picks, "groups": groups, "kept": kept, "dtype": dtype,
            "sigmoid": sigmoid, "bias": bias, "renormalize": renormalize, "masked": masked, "grad": grad, "scaling": scaling}


def listed():
    return [
        # activations of a decode batch, shared by several projections
        _quantize("quantize_bf16_32x7168", 32, 7168, "bf16"),
        # activations of a long prompt
        _quantize("quantize_fp16_8191x14336", 8191, 14336, "fp16"),
        # decode of one token through a small projection: launch latency counts
        _linear("linear_bf16_512x7168_t1", 512, 7168, 1, "bf16"),
        # a decode batch of sixteen through a large feed-forward matrix
        _linear("linear_fp16_28672x8192_t16", 28672, 8192, 16, "fp16"),
        # an odd batch with a bias
        _linear("linear_bf16_13824x5120_t100", 13824, 5120, 100, "bf16", True),
        # a long prompt
        _linear("linear_bf16_8192x8192_t4000", 8192, 8192, 4000, "bf16"),
        # one token through an expert layer
        _experts("experts_bf16_8_t1", _MOE[0], 1, "bf16"),
        # a decode batch through many small experts, half of which another card holds
        _experts("experts_fp16_128_t50_held64", _MOE[1], 50, "fp16", 64),
        # a prompt through a few large experts
        _experts("experts_bf16_8_t1000", _MOE[0], 1000, "bf16"),
        # the router of a decode step: grouped experts, fp32 logits, sigmoid scores, a bias that balances, padded rows
        _routing("routing_fp32_e256_t16", 16, _ROUTERS[3], "fp32", True, True, True, True, False, 2.5),
        # a training step's router, softmax over bf16 logits
        _routing("routing_bf16_e64_t16384", 16384, _ROUTERS[1], "bf16"),
        # a training step's grouped router in fp32 with sigmoid scores, a bias and padded tokens
        _routing("routing_fp32_e256_t8191", 8191, _ROUTERS[3], "fp32", True, True, True, True, True, 2.5),
    ]


def _log_int(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(max(low, high))))))


def draw(rng):
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= _MAX_BYTES and w["flops"] <= _MAX_FLOPS:
            return case


def _draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "linear", "experts", "experts", "routing", "routing"])
    dtype = rng.choice(["bf16", "fp16"])
    if kind == "quantize":
        case = _quantize("", _log_int(rng, 1, 16384), 128 * _log_int(rng, 1, 148), rng.choice(["bf16", "fp16", "fp32"]))
    elif kind == "linear":
        rows, k = rng.choice(_SHAPES)
        if rng.random() < 0.5:
            rows, k = 16 * _log_int(rng, 8, 1792), 128 * _log_int(rng, 3, 64)
        tokens = 1 if rng.random() < 0.2 else _log_int(rng, 2, min(8192, _MAX_FLOPS / (2 * rows * k)))
        case = _linear("", rows, k, tokens, dtype, rng.random() < 0.3)
    elif kind == "experts":
        layer = rng.choice(_MOE)
        if rng.random() < 0.4:
            e = _log_int(rng, 4, 160)
            layer = (e, rng.randint(1, min(8, e)), 128 * _log_int(rng, 4, 32), 128 * _log_int(rng, 2, 16))
        e, picks, hidden, inter = layer
        tokens = _log_int(rng, 1, min(2048, _MAX_PLAIN / (6 * e * hidden * inter)))
        case = _experts("", layer, tokens, dtype, None if rng.random() < 0.7 else rng.randint(1, e))
    else:
        router = rng.choice(_ROUTERS)
        if rng.random() < 0.4:
            e = rng.randint(2, 512)
            router = (e, rng.randint(1, min(10, e)), 1, 1)
        case = _routing("", _log_int(rng, 1, 16384), router, rng.choice(["bf16", "fp16", "fp32"]), rng.random() < 0.5, rng.random() < 0.5,
                        rng.random() < 0.7, rng.random() < 0.4, rng.random() < 0.7, rng.choice([1.0, 2.5]))
    case.pop("name")
    return case


# ------------------------------------------------------------------------------------------------------------ inputs
def _activations(gen, tokens, k, dtype):
    """Normal values, some columns larger than others, as behind a norm."""
    x = torch.randn((tokens, k), generator=gen, device="cuda")
    return (x * torch.exp(0.5 * torch.randn(k, generator=gen, device="cuda"))).to(dtype)


def _weights(gen, rows, k):
    """Codes of normal weights as a checkpoint has them, [rows, k], and the largest magnitude of a 128 x 128 block over 448."""
    w = torch.randn((rows, k), generator=gen, device="cuda") * k ** -0.5
    full = torch.zeros(((rows + 127) // 128 * 128, k), device="cuda")
    full[:rows] = w.abs()
    scale = full.view(-1, 128, k // 128, 128).amax(dim=(1, 3)) / 448
    del full
    return (w / scale.repeat_interleave(128, 0)[:rows].repeat_interleave(128, 1)).to(_E4M3), scale


def _expert_weights(gen, rows, k, held):
    codes = torch.empty((held, rows, k), dtype=_E4M3, device="cuda")
    scales = torch.empty((held, rows // 128, k // 128), device="cuda")
    for e in range(held):
        codes[e], scales[e] = _weights(gen, rows, k)
    return codes, scales


def _popular(gen, tokens, experts):
    """Router logits, some experts more popular than others."""
    return torch.randn((tokens, experts), generator=gen, device="cuda") + 0.5 * torch.randn(experts, generator=gen, device="cuda")


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    kind, tokens, dtype = case["kind"], case["tokens"], _DTYPE[case["dtype"]]
    state = {"kind": kind, "case": case}
    if kind == "quantize":
        state["x"] = _activations(gen, tokens, case["k"], dtype)
    elif kind == "linear":
        state["w"] = _weights(gen, case["rows"], case["k"])
        state["x"] = _activations(gen, tokens, case["k"], dtype)
        state["bias"] = torch.randn((1, case["rows"]), generator=gen, device="cuda").to(dtype) if case["bias"] else None
    elif kind == "experts":
        e, held, hidden, inter = case["experts"], case["held"], case["hidden"], case["inter"]
        state["w1"], state["w2"] = _expert_weights(gen, 2 * inter, hidden, held), _expert_weights(gen, hidden, inter, held)
        state["x"] = _activations(gen, tokens, hidden, dtype)
        logits = _popular(gen, tokens, e)
        state["ids"] = torch.sort(logits, dim=-1, descending=True, stable=True)[1][:, :case["picks"]].to(torch.int32).contiguous()
        p = torch.gather(torch.exp(logits), 1, state["ids"].long())
        state["weights"] = (p / p.sum(dim=-1, keepdim=True)).to(dtype)
        state["map"] = None
        if held < e:
            state["map"] = torch.full((e,), -1, dtype=torch.int32, device="cuda")
            here = torch.randperm(e, generator=gen, device="cuda")[:held].sort()[0]
            state["map"][here] = torch.arange(held, dtype=torch.int32, device="cuda")
    else:
        state["logits"] = _popular(gen, tokens, case["experts"]).to(dtype).requires_grad_(case["grad"])
        state["bias"] = 0.1 * torch.randn(case["experts"], generator=gen, device="cuda") if case["bias"] else None
        state["mask"] = torch.rand(tokens, generator=gen, device="cuda") < 0.8 if case["masked"] else None
        # fp16 gradients come of a scaled loss, as in a training program in fp16
        state["up"] = (torch.randn((tokens, case["picks"]), generator=gen, device="cuda") * (64 if case["dtype"] == "fp16" else 1)).to(dtype)
    if own:
        # what a program keeps of its weights: the library's layout, packed once at load time, in place of the checkpoint's rows
        import muxi_layout_kernels as mlk
        for name in ("w", "w1", "w2"):
            if name in state:
                codes, scale = state[name]
                state[name] = mlk.pack_layout_a(codes), scale
    return state


# -------------------------------------------------------------------------------------------------------- plain forms
def _plain_quantize(x):
    """codes [T, K], scales [T, K / 128]"""
    x = x.float().unflatten(-1, (-1, 128))
    most = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(dim=-1)
    m, e = torch.frexp(most)                                                 # most = m 2^e, 448 = 0.875 2^9
    e = torch.where(most > 0, e - torch.where(m <= 0.875, 9, 8), -100).clamp(min=-100)
    scale, inverse = (((s * e + 127) << 23).to(torch.int32).view(torch.float32) for s in (1, -1))
    codes = (x * inverse.unsqueeze(-1)).to(_E4M3)
    return codes.flatten(-2), scale


def _rounded(x):
    """fp32 activations as their codes stand for them"""
    codes, scale = _plain_quantize(x)
    return (codes.float().unflatten(-1, (-1, 128)) * scale.unsqueeze(-1)).flatten(-2)


def _dequantised(codes, scale):
    rows, k = codes.shape[-2:]
    return codes.float() * scale.repeat_interleave(128, -2)[..., :rows, :].repeat_interleave(128, -1)


def _plain_linear(state):
    y = _rounded(state["x"]) @ _dequantised(*state["w"]).t()
    if state["bias"] is not None:
        y = y + state["bias"].float()
    return y.to(state["x"].dtype)


def _plain_experts(state):
    x, ids, held = _rounded(state["x"]), state["ids"].long(), state["case"]["held"]
    if state["map"] is not None:
        ids = state["map"].long()[ids]
    w1, w2 = state["w1"], state["w2"]
    share = state["weights"].float().unsqueeze(-1) * (ids.unsqueeze(-1) == torch.arange(held, device=x.device))
    share = share.sum(dim=1)                                                 # [tokens, held]
    if x.shape[0] == 1 and ids.shape[1] < held:                              # one token: only its experts' weights are read
        ids = ids.clamp(min=0)[0]
        w1, w2 = (tuple(p.view(torch.uint8)[ids].view(p.dtype) if p.dtype == _E4M3 else p[ids] for p in w) for w in (w1, w2))
        share = share[:, ids]
    w1, w2 = _dequantised(*w1), _dequantised(*w2)                            # [e, 2 I, H], [e, H, I]
    e, hidden, inter = w2.shape
    gate, up = (x @ w1.reshape(e * 2 * inter, hidden).t()).view(-1, e, 2, inter).unbind(2)
    h = _rounded(gate / (1 + torch.exp(-gate)) * up) * share.unsqueeze(-1)
    return (h.reshape(-1, e * inter) @ w2.transpose(1, 2).reshape(e * inter, hidden)).to(state["x"].dtype)


def _plain_selection(state, x):
    """The experts of each token, [tokens, picks].  Logits are compared as they are; scores and biases in 64 bits, where neighbours keep their order."""
    c = state["case"]
    tokens, experts = x.shape
    rank = x
    if state["bias"] is not None:
        s = x.double()
        s = 1 / (1 + torch.exp(-s)) if c["sigmoid"] else torch.exp(s - s.max(dim=-1, keepdim=True)[0])
        rank = (s if c["sigmoid"] else s / s.sum(dim=-1, keepdim=True)) + state["bias"].double()
    if c["groups"] > 1:
        each = rank.view(tokens, c["groups"], -1)
        best = torch.sort(each, dim=-1, descending=True)[0]
        best = best[..., 0] if state["bias"] is None else best[..., :2].sum(dim=-1)
        kept = torch.sort(best, dim=-1, descending=True, stable=True)[1][:, :c["kept"]]
        keep = (kept.unsqueeze(-1) == torch.arange(c["groups"], device=x.device)).any(dim=1)
        rank = torch.where(keep.unsqueeze(-1), each, -math.inf).view(tokens, experts)
    return torch.sort(rank, dim=-1, descending=True, stable=True)[1][:, :c["picks"]]


def _plain_routing(state):
    c, x, mask = state["case"], state["logits"].detach().float(), state["mask"]
    ids = _plain_selection(state, x)
    score = 1 / (1 + torch.exp(-x)) if c["sigmoid"] else torch.exp(x - x.max(dim=-1, keepdim=True)[0])
    if not c["sigmoid"]:
        score = score / score.sum(dim=-1, keepdim=True)
    p = torch.gather(score, 1, ids)
    total = p.sum(dim=-1, keepdim=True)
    w = p / total if c["renormalize"] else p
    valid = 1.0 if mask is None else mask.float().unsqueeze(-1)
    out_ids = ids if mask is None else torch.where(mask.unsqueeze(-1), ids, -1)
    out = [out_ids.to(torch.int32), (w * c["scaling"] * valid).to(state["logits"].dtype)]
    if c["grad"]:
        g = state["up"].float() * c["scaling"] * valid
        dp = (g - (g * w).sum(dim=-1, keepdim=True)) / total if c["renormalize"] else g      # of the picks' scores
        if c["sigmoid"]:
            dx = torch.zeros_like(x).scatter(1, ids, dp * p * (1 - p))
        elif c["renormalize"]:
            dx = torch.zeros_like(x).scatter(1, ids, dp * p)                                 # sum of dp p is 0
        else:
            dx = torch.zeros_like(x).scatter(1, ids, dp * p) - score * (dp * p).sum(dim=-1, keepdim=True)
        out.append(dx.to(state["logits"].dtype))
    return out


def run(state):
    kind, c = state["kind"], state["case"]
    if own:
        import muxi_layout_kernels as mlk
        if kind == "quantize":
            return mlk.quantize_fp8(state["x"])
        if kind == "linear":
            w, scale = state["w"]
            return mlk.gemm_layoutA_fp8(w, scale, state["x"], bias=state["bias"])
        if kind == "experts":
            (w1, s1), (w2, s2) = state["w1"], state["w2"]
            return mlk.fused_experts_fp8(state["x"], w1, w2, state["ids"], state["weights"], s1, s2, experts_map=state["map"])
        ids, w = mlk.moe_routing(state["logits"], c["picks"], "sigmoid" if c["sigmoid"] else "softmax", c["renormalize"], c["groups"], c["kept"],
                                 gating_bias=state["bias"], scaling=c["scaling"], token_mask=state["mask"])
        if not c["grad"]:
            return [ids, w]
        grad, = torch.autograd.grad(w, state["logits"], grad_outputs=state["up"])
        return [ids, w.detach(), grad]
    if kind == "quantize":
        return _plain_quantize(state["x"])
    if kind == "linear":
        return _plain_linear(state)
    if kind == "experts":
        return _plain_experts(state)
    return _plain_routing(state)


# --------------------------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    """Weights, scales and activations read once, outputs written once; two operations per weight and token.  Of an expert layer, the experts
    that even routing would be expected to reach and the pairs that stay on this card.  Of the routing, the logits read (again for the gradient) and their
    gradient written, some ten operations each; the picks, the bias and the mask."""
    tokens, size = case["tokens"], 4 if case["dtype"] == "fp32" else 2

    def matrix(rows, k):
        return rows * k + 4 * ((rows + 127) // 128) * (k // 128)

    if case["kind"] == "quantize":
        n = tokens * case["k"]
        return {"bytes": (size + 1) * n + 4 * (n // 128), "flops": 3 * n}
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
    small = (4 + size) * tokens * picks + (tokens if case["masked"] else 0) + (4 * e if case["bias"] else 0)
    passes = 3 if case["grad"] else 1
    return {"bytes": passes * size * tokens * e + small * (2 if case["grad"] else 1), "flops": 10 * passes * tokens * e}


# ------------------------------------------------------------------------------------------------- the definition in 64 bits
def _inputs(case, seed):
    """The inputs of `prepare` as a plain program has them."""
    global own
    was, own = own, False
    try:
        return prepare(case, seed)
    finally:
        own = was


def _two_to(e):
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _quantize64(x):
    """(values of the codes [T, K], scales [T, K / 128]), from the steps of the format: 2^(exponent - 3), 2^-9 at least."""
    blocks = x.double().view(x.shape[0], -1, 128)
    most = torch.nan_to_num(blocks, nan=0.0, posinf=0.0, neginf=0.0).abs().max(dim=-1)[0]
    e = torch.full_like(most, -100.0)
    for up in range(-100, 129):                                              # the smallest power of two that is large enough
        e = torch.where(most > 448.0 * 2.0 ** up, float(up + 1), e)
    scale = _two_to(e)
    v = blocks / scale.unsqueeze(-1)
    step = torch.floor(torch.log2(v.abs().clamp(min=2.0 ** -6)))
    step = _two_to(torch.where(v.abs() >= _two_to(step + 1), step + 1, torch.where(v.abs().clamp(min=2.0 ** -6) < _two_to(step), step - 1, step)) - 3)
    return (torch.round(v / step) * step).view(x.shape), scale


def _rounded64(x):
    values, scale = _quantize64(x)
    return values * scale.repeat_interleave(128, dim=-1)


def _table64(codes, scale):
    """Every weight from the table of the 256 values of a code."""
    b = torch.arange(256, device="cuda")
    exponent, mantissa = (b >> 3) & 15, (b & 7).double()
    table = torch.where(exponent > 0, (1 + mantissa / 8) * _two_to(exponent - 7), mantissa * 2.0 ** -9) * torch.where(b >= 128, -1.0, 1.0)
    rows, k = codes.shape
    out = table[codes.view(torch.uint8).int()]
    for i in range(0, rows, 128):
        out[i:i + 128].view(-1, k // 128, 128).mul_(scale[i // 128].double().view(1, -1, 1))
    return out


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        return _quantize64(s["x"])
    if kind == "linear":
        out = torch.nn.functional.linear(_rounded64(s["x"]), _table64(*s["w"]))
        return out if s["bias"] is None else out + s["bias"].double()
    if kind == "experts":
        x, out = _rounded64(s["x"]), torch.zeros(s["x"].shape, dtype=torch.float64, device="cuda")
        for e in range(case["held"]):
            hit = (s["ids"] if s["map"] is None else s["map"][s["ids"].long()]) == e
            token, pick = hit.nonzero(as_tuple=True)
            if token.numel():
                both = torch.nn.functional.linear(x[token], _table64(s["w1"][0][e], s["w1"][1][e]))
                h = _rounded64(torch.nn.functional.silu(both[:, :case["inter"]]) * both[:, case["inter"]:])
                out.index_add_(0, token, torch.nn.functional.linear(h, _table64(s["w2"][0][e], s["w2"][1][e])) * s["weights"][token, pick].double().unsqueeze(1))
        return out
    # routing: weights by torch's own functions in 64 bits, the gradient by its differentiation
    leaf = s["logits"].detach().double().requires_grad_(True)
    score = torch.sigmoid(leaf) if case["sigmoid"] else torch.softmax(leaf, dim=-1)
    with torch.no_grad():
        rank = leaf if s["bias"] is None else score + s["bias"].double()
        if case["groups"] > 1:
            each = rank.view(case["tokens"], case["groups"], -1)
            best = each.topk(1 if s["bias"] is None else 2, dim=-1)[0].sum(dim=-1)
            order = torch.argsort(-best, dim=-1, stable=True)
            drop = torch.zeros_like(best, dtype=torch.bool).scatter(1, order[:, case["kept"]:], True)
            rank = each.masked_fill(drop.unsqueeze(-1), -math.inf).flatten(1)
        ids = torch.argsort(-rank, dim=-1, stable=True)[:, :case["picks"]]
    w = score.gather(1, ids)
    if case["renormalize"]:
        w = w / w.sum(dim=-1, keepdim=True)
    w = w * case["scaling"]
    if s["mask"] is not None:
        w = w * s["mask"].unsqueeze(-1)
    if not case["grad"]:
        return [None, w.detach()]
    grad, = torch.autograd.grad(w, leaf, grad_outputs=s["up"].double())
    return [None, w.detach(), grad]
