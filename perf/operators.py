"""Cases of the 4-bit products and of the token shuffle around routed experts, for timing and for comparing them with
their plain forms.

    linear    y [T, rows] = x [T, cols] W^T, W[r, c] = (code[r, c] - zero[r, g]) scale[r, g], g = c // group, the codes
              4 bits wide: a replica's projection in 4 bits, on a decode step's or a draft pass's tokens
    experts   the same product for routed experts: row p of the output is the token of the p-th pair of the sorted
              order times that pair's expert; gated: silu(gate) * up of the expert's two halves
    shuffle   tokens sorted by expert and back: the order, x's rows in that order, the weighted sums of the experts'
              rows, and with train the gradients of x, of the experts' rows and of the routing weights

`own` chooses between the plain form (elementary torch operations in 32 bits, rounded once) and the package's calls.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}

# What a drawn case may cost at most: the listed cases' largest products and token matrices.
MOST_WEIGHTS = 28672 * 4096
MOST_PRODUCT = 28672 * 4096 * 272
MOST_EXPERT_WEIGHTS = 128 * 1536 * 2048
MOST_EXPERT_PRODUCT = 2048 * 8 * 1536 * 2048
MOST_ROWS = 8192 * 8 * 2048


def listed():
    def linear(name, tokens, rows, cols, group, zeros, dtype):
        return {"name": name, "op": "linear", "tokens": tokens, "rows": rows, "cols": cols, "group": group,
                "zeros": zeros, "dtype": dtype}

    def experts(name, tokens, experts, topk, hidden, inter, gated, group, zeros, dtype):
        return {"name": name, "op": "experts", "tokens": tokens, "experts": experts, "topk": topk, "hidden": hidden,
                "inter": inter, "gated": gated, "group": group, "zeros": zeros, "dtype": dtype}

    def shuffle(name, tokens, experts, topk, hidden, train, dtype, nowhere):
        return {"name": name, "op": "shuffle", "tokens": tokens, "experts": experts, "topk": topk, "hidden": hidden,
                "train": train, "dtype": dtype, "nowhere": nowhere}

    return [
        # The k (or v) projection of the Llama-3-8B shape on one token of one sequence: the smallest call, all latency.
        linear("linear k 1 token", 1, 1024, 4096, 128, False, "bf16"),
        # The down projection on one token, f16 with zero points and small groups, as weights quantised elsewhere come.
        linear("linear down 1 token f16", 1, 4096, 14336, 64, True, "f16"),
        # The gate and up projections on one sequence's draft pass of 16 + 1 tokens.
        linear("linear gate_up 17 tokens", 17, 28672, 4096, 128, False, "bf16"),
        # The same module on 16 sequences' draft passes: the framework's headline batch.
        linear("linear gate_up 272 tokens", 272, 28672, 4096, 128, False, "bf16"),
        # A ragged module (a row slice of the 27648 x 5120 projection, columns no multiple of 8), the finest groups.
        linear("linear ragged 33 tokens", 33, 6913, 5119, 32, True, "bf16"),
        # Gate and up of the 128-expert layer for one decoded token: eight experts of one row each.
        experts("experts gate_up 1 token", 1, 128, 8, 2048, 768, True, 128, False, "bf16"),
        # Its down projection on 272 draft tokens: 17 rows an expert, every expert's weights read.
        experts("experts down 272 tokens", 272, 128, 8, 2048, 768, False, 32, True, "f16"),
        # Gate and up on a calibration or prefill sequence of 2048 tokens.
        experts("experts gate_up 2048 tokens", 2048, 128, 8, 2048, 768, True, 128, False, "bf16"),
        # One decoded token on its way to the experts and back.
        shuffle("shuffle 1 token", 1, 128, 8, 2048, False, "bf16", 0.0),
        # A draft pass's tokens, some of them padding that is routed nowhere.
        shuffle("shuffle 272 tokens", 272, 128, 8, 2048, False, "bf16", 0.05),
        # A training step over an odd number of tokens, in 32 bits.
        shuffle("shuffle train 1023 f32", 1023, 60, 4, 1408, True, "f32", 0.0),
        # A training step over four sequences of 2048 tokens.
        shuffle("shuffle train 8192", 8192, 128, 8, 2048, True, "bf16", 0.0),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["linear", "linear", "experts", "shuffle"])
    if op == "linear":
        rows, cols = _log(rng, 256, 28672), _log(rng, 256, 14336)
        if rng.random() < 0.7:                       # most modules have columns in multiples of 8
            cols = cols // 8 * 8
        rows = min(rows, MOST_WEIGHTS // cols)
        tokens = _log(rng, 1, 272)
        return {"op": op, "tokens": tokens, "rows": rows, "cols": cols, "group": rng.choice([32, 64, 128]),
                "zeros": rng.random() < 0.5, "dtype": rng.choice(["bf16", "f16"])}
    if op == "experts":
        hidden, inter = 8 * _log(rng, 32, 256), 8 * _log(rng, 16, 96)
        experts = _log(rng, 8, 128)
        topk = rng.randint(1, 8)
        tokens = _log(rng, 1, 2048)
        tokens = max(1, min(tokens, MOST_EXPERT_PRODUCT // (topk * 2 * inter * hidden)))
        return {"op": op, "tokens": tokens, "experts": experts, "topk": topk, "hidden": hidden, "inter": inter,
                "gated": rng.random() < 0.5, "group": rng.choice([32, 64, 128]), "zeros": rng.random() < 0.5,
                "dtype": rng.choice(["bf16", "f16"])}
    hidden, topk = _log(rng, 64, 4096), rng.randint(1, 8)
    experts = _log(rng, 8, 256)
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    tokens = max(1, min(_log(rng, 1, 8192), MOST_ROWS // (topk * hidden) // (2 if dtype == "f32" else 1)))
    return {"op": op, "tokens": tokens, "experts": experts, "topk": topk, "hidden": hidden,
            "train": rng.random() < 0.5, "dtype": dtype, "nowhere": rng.choice([0.0, 0.05])}


def work(case):
    size = 4 if case["dtype"] == "f32" else 2
    T = case["tokens"]
    if case["op"] == "linear":
        rows, cols = case["rows"], case["cols"]
        groups = -(-cols // case["group"])
        weights = rows * cols / 2 + rows * groups * (2 + (0.5 if case["zeros"] else 0))
        return {"bytes": weights + size * T * (rows + cols), "flops": 2 * T * rows * cols}
    H, K = case["hidden"], case["topk"]
    P = T * K
    if case["op"] == "experts":
        E, R = case["experts"], case["inter"]
        rows, cols = (2 * R, H) if case["gated"] else (H, R)
        used = E * (1 - (1 - min(K, E) / E) ** T)    # the experts that some token reaches, whose weights are read
        groups = -(-cols // case["group"])
        weights = used * (rows * cols / 2 + rows * groups * (2 + (0.5 if case["zeros"] else 0)))
        x = T * H if case["gated"] else P * R
        return {"bytes": weights + size * (x + P * (R if case["gated"] else H)), "flops": 2 * P * rows * cols}
    P = int(P * (1 - case["nowhere"]))
    ids = T * K * (4 + 4 + 4 + 4)                    # ids and weights read, order and where written
    forward = size * (T * H + P * H + P * H + T * H) + ids
    if not case["train"]:
        return {"bytes": forward, "flops": 2 * P * H}
    # the incoming gradients of the sorted rows and of the sums read, those of x, the rows and the weights written
    return {"bytes": forward + size * (P * H + T * H + T * H + P * H) + 4 * T * K, "flops": 6 * P * H}


# --- inputs ----------------------------------------------------------------------------------------------------------


def _quantised(shape, group, zeros, dtype, g):
    """(codes [.., ceil(cols / 2)] uint8, scales [.., groups], zeros [.., groups] uint8 or None) of weights N(0, 0.02)
    of `shape`, each group of `group` columns spanning its own range."""
    lead, cols = shape[:-1], shape[-1]
    groups = -(-cols // group)
    w = torch.randn(*lead, groups, group, generator=g, device="cuda").mul_(0.02)
    if groups * group > cols:                        # the columns that the last group lacks
        w[..., -1, cols - (groups - 1) * group:] = 0
    if zeros:
        lo, hi = w.amin(-1).clamp_(max=0), w.amax(-1).clamp_(min=0)
        scales = ((hi - lo) / 15).clamp_(min=1e-6).to(dtype)
        zero = (-lo / scales.float()).round_().clamp_(0, 15)
    else:
        scales = (w.abs().amax(-1) / 7).clamp_(min=1e-6).to(dtype)
        zero = torch.full_like(scales, 8, dtype=torch.float32)
    q = w.div_(scales.float().unsqueeze(-1)).round_().add_(zero.unsqueeze(-1)).clamp_(0, 15).to(torch.uint8)
    q = q.reshape(*lead, groups * group)
    even, odd = q[..., 0:cols:2], q[..., 1:cols:2]
    codes = even.clone()
    codes[..., : odd.shape[-1]] |= odd << 4
    return codes, scales, zero.to(torch.uint8) if zeros else None


def _activations(tokens, cols, dtype, g):
    """Rows of N(0, 1) with a lognormal scale for each channel, as hidden states have."""
    x = torch.randn(tokens, cols, generator=g, device="cuda")
    return (x * torch.exp(0.5 * torch.randn(cols, generator=g, device="cuda"))).to(dtype)


def _routing(tokens, experts, topk, nowhere, g):
    """(ids [T, K] int32, weights [T, K] f32): the top-k experts of random router logits, weights of a softmax over
    them, the share `nowhere` of the tokens routed nowhere (-1)."""
    topk = min(topk, experts)
    logits = torch.randn(tokens, experts, generator=g, device="cuda")
    top, ids = logits.topk(topk, dim=-1)
    weights = torch.exp(top - top[:, :1])
    weights = weights / weights.sum(-1, keepdim=True)
    gone = torch.rand(tokens, generator=g, device="cuda") < nowhere
    return torch.where(gone[:, None], -1, ids).to(torch.int32), weights.float()


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    T = case["tokens"]
    s = {"op": case["op"], "dtype": dtype}
    if case["op"] == "linear":
        rows, cols, group = case["rows"], case["cols"], case["group"]
        s["codes"], s["scales"], s["zeros"] = _quantised((rows, cols), group, case["zeros"], dtype, g)
        s.update(x=_activations(T, cols, dtype, g), cols=cols, group=group)
        if own:                                      # the module's weights, laid out once at load
            from p2pllm_b200 import compact
            s["tiles"] = compact.Tiles([("int4", s["codes"], s["scales"], s["zeros"], cols, group)])
        return s
    E, H = case["experts"], case["hidden"]
    ids, weights = _routing(T, E, case["topk"], case.get("nowhere", 0.0), g)
    P = ids.numel()
    s.update(ids=ids, experts=E)
    if case["op"] == "experts":
        R, gated, group = case["inter"], case["gated"], case["group"]
        rows, cols = (2 * R, H) if gated else (H, R)
        s["codes"], s["scales"], s["zeros"] = _quantised((E, rows, cols), group, case["zeros"], dtype, g)
        # gated products read the tokens' rows, the down products rows that are in the experts' order already
        s.update(x=_activations(T if gated else P, cols, dtype, g), gated=gated, cols=cols, group=group)
        s["most"] = int(torch.bincount(ids.reshape(-1), minlength=E).max())
        if own:                                      # the layer's weights, and the order that the step before made
            from p2pllm_b200 import moe
            s["tiles"] = moe.Int4Experts([("int4", s["codes"], s["scales"], s["zeros"], cols, group)], gated=gated)
            s["order"] = moe.sort_tokens(ids, E)
        return s
    s.update(x=torch.randn(T, H, generator=g, device="cuda").to(dtype), weights=weights, train=case["train"],
             y=torch.randn(P, H, generator=g, device="cuda").to(dtype))
    if case["train"]:
        s["grad_sorted"] = torch.randn(P, H, generator=g, device="cuda").to(dtype)
        s["grad_out"] = torch.randn(T, H, generator=g, device="cuda").to(dtype)
        used = int((ids >= 0).sum())
        s["grad_sorted"][used:] = 0
        for name in ("x", "y", "weights"):
            s[name].requires_grad_(True)
    return s


# --- one pass --------------------------------------------------------------------------------------------------------


def run(s):
    if own:
        return _run_own(s)
    with torch.no_grad():
        return {"linear": _plain_linear, "experts": _plain_experts, "shuffle": _plain_shuffle}[s["op"]](s)


def _run_own(s):
    from p2pllm_b200 import moe
    if s["op"] == "linear":
        return s["tiles"](s["x"])
    if s["op"] == "experts":
        return s["tiles"](s["x"], s["order"], gather=s["gated"])
    order = moe.sort_tokens(s["ids"], s["experts"])
    xs = moe.to_experts(s["x"], order)
    out = moe.from_experts(s["y"], order, s["weights"])
    got = {"order": order.order, "where": order.where, "offsets": order.offsets, "sorted": xs, "out": out}
    if s["train"]:
        got["dx"], got["dy"], got["dweights"] = torch.autograd.grad(
            (xs, out), (s["x"], s["y"], s["weights"]), (s["grad_sorted"], s["grad_out"]))
        got["sorted"], got["out"] = xs.detach(), out.detach()
    return got


def _dense(s, experts=None):
    """The weights that the codes stand for, in 32 bits; of routed experts only `experts`, if given."""
    codes, scales, zeros = (t if t is None or experts is None else t[experts] for t in (s["codes"], s["scales"], s["zeros"]))
    group, cols = s["group"], s["cols"]
    q = torch.stack((codes & 15, codes >> 4), dim=-1).flatten(-2)[..., :cols].float()
    zero = 8.0 if zeros is None else zeros.float().repeat_interleave(group, -1)[..., :cols]
    return (q - zero) * scales.float().repeat_interleave(group, -1)[..., :cols]


def _plain_linear(s):
    return (s["x"].float() @ _dense(s).mT).to(s["dtype"])


def _order(ids, experts):
    """(order, where, offsets) of the pairs sorted by expert, pairs of one expert in their own order; -1 behind the
    last pair and for a pair that is routed nowhere."""
    flat = ids.reshape(-1).long()
    routed = flat >= 0
    key = torch.where(routed, flat, experts)
    order = torch.sort(key, stable=True).indices
    where = torch.empty_like(order)
    where[order] = torch.arange(order.numel(), device=order.device)
    counts = torch.zeros(experts + 1, dtype=torch.int64, device=flat.device).index_add_(0, key, torch.ones_like(key))
    offsets = torch.zeros_like(counts)
    offsets[1:] = counts[:-1].cumsum(0)
    order = torch.where(torch.arange(order.numel(), device=order.device) < offsets[-1], order, -1)
    return order, torch.where(routed, where, -1), offsets


def _plain_experts(s):
    ids, E, x, most = s["ids"], s["experts"], s["x"].float(), s["most"]
    order, _, offsets = _order(ids, E)
    if s["gated"]:
        x = x[order // ids.shape[1]]
    expert = ids.reshape(-1).long()[order]
    if order.numel() <= E:                           # few rows: each with its own expert's weights
        y = torch.bmm(x.unsqueeze(1), _dense(s, expert).mT).squeeze(1)
    else:                                            # each expert's rows padded to the most that one has
        slot = torch.arange(order.numel(), device=x.device) - offsets[expert]
        padded = torch.zeros(E, most, x.shape[1], device=x.device)
        padded[expert, slot] = x
        y = torch.bmm(padded, _dense(s).mT)[expert, slot]
    if s["gated"]:
        gate, up = y.chunk(2, dim=-1)
        y = gate / (1 + torch.exp(-gate)) * up
    return y.to(s["dtype"])


def _plain_shuffle(s):
    ids, x, y, w = s["ids"], s["x"], s["y"], s["weights"]
    T, K = ids.shape
    order, where, offsets = _order(ids, s["experts"])
    live = (order >= 0)[:, None]
    here = (where >= 0).view(T, K, 1)
    at = where.clamp(min=0)
    xs = torch.where(live, x[order.clamp(min=0) // K], 0)
    rows = torch.where(here, y[at].float().view(T, K, -1), 0)
    out = (w.unsqueeze(-1) * rows).sum(1).to(x.dtype)
    got = {"order": order.int(), "where": where.int(), "offsets": offsets.int(), "sorted": xs, "out": out}
    if s["train"]:
        gout = s["grad_out"].float()
        got["dx"] = torch.where(here, s["grad_sorted"][at].float().view(T, K, -1), 0).sum(1).to(x.dtype)
        back = w.reshape(-1)[order.clamp(min=0), None] * gout[order.clamp(min=0) // K]
        got["dy"] = torch.where(live, back, 0).to(y.dtype)
        got["dweights"] = (rows * gout.unsqueeze(1)).sum(-1)
    return got


# --- the definition in 64 bits ---------------------------------------------------------------------------------------


def _exact_weights(codes, scales, zeros, cols, group):
    low, high = torch.bitwise_and(codes, 0x0F), torch.bitwise_right_shift(codes, 4)
    w = torch.zeros(codes.shape[0], 2 * codes.shape[1], dtype=torch.float64, device=codes.device)
    w[:, 0::2], w[:, 1::2] = low.double(), high.double()
    w = w[:, :cols]
    for k in range(scales.shape[1]):
        part = w[:, k * group:(k + 1) * group]
        part -= 8.0 if zeros is None else zeros[:, k:k + 1].double()
        part *= scales[:, k:k + 1].double()
    return w


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "linear":
        w = _exact_weights(s["codes"], s["scales"], s["zeros"], s["cols"], s["group"])
        return torch.einsum("tc,rc->tr", s["x"].double(), w)
    flat = s["ids"].reshape(-1).tolist()
    K = s["ids"].shape[1]
    by_expert = [[] for _ in range(case["experts"])]
    for pair, e in enumerate(flat):
        if e >= 0:
            by_expert[e].append(pair)
    order = [pair for pairs in by_expert for pair in pairs]
    if case["op"] == "experts":
        x, out, at = s["x"].double(), [], 0
        for e, pairs in enumerate(by_expert):
            if not pairs:
                continue
            zeros = None if s["zeros"] is None else s["zeros"][e]
            w = _exact_weights(s["codes"][e], s["scales"][e], zeros, s["cols"], s["group"])
            rows = x[[p // K for p in pairs]] if s["gated"] else x[at:at + len(pairs)]
            y = rows @ w.T
            if s["gated"]:
                R = y.shape[1] // 2
                y = y[:, :R] * torch.sigmoid(y[:, :R]) * y[:, R:]
            out.append(y)
            at += len(pairs)
        return torch.cat(out)
    T, H = s["x"].shape
    dev = s["x"].device
    with torch.no_grad():
        x, y, w = s["x"].double(), s["y"].double(), s["weights"].double()
        pairs = torch.tensor(order, dtype=torch.long, device=dev)
        token, n = pairs // K, len(order)
        xs = torch.zeros(T * K, H, dtype=torch.float64, device=dev)
        xs[:n] = x[token]
        out = torch.zeros(T, H, dtype=torch.float64, device=dev)
        out.index_add_(0, token, w.reshape(-1)[pairs, None] * y[:n])
        got = {"order": None, "where": None, "offsets": None, "sorted": xs, "out": out}
        if case["train"]:
            gout = s["grad_out"].double()
            got["dx"] = torch.zeros_like(x).index_add_(0, token, s["grad_sorted"][:n].double())
            got["dy"] = torch.zeros_like(y)
            got["dy"][:n] = w.reshape(-1)[pairs, None] * gout[token]
            got["dweights"] = torch.zeros_like(w.reshape(-1))
            got["dweights"][pairs] = (gout[token] * y[:n]).sum(-1)
            got["dweights"] = got["dweights"].view(T, K)
    return got
