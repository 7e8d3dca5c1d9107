"""Timed cases of the router's balance loss with its counts and gradient, the products with 4-bit
weights (one matrix, and one matrix per expert), the 4-bit quantisation of weights and back, and the
layer norm before a block with its gradients.

``run`` makes the framework's calls where ``own`` is true; elsewhere it computes the same results
with elementary torch operations in 32 bits. ``exact`` computes them from the definitions in 64
bits.
"""
import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # a micro-batch of a fine-tuning step: 64 tokens over 256 experts, top 8
        {"name": "balance micro", "op": "balance", "tokens": 64, "experts": 256, "top_k": 8,
         "sequences": 0, "scoring": "softmax", "dtype": "fp32", "grad": True},
        # packed sequences with padding behind the last, an odd number of tokens, 16-bit logits
        {"name": "balance packed", "op": "balance", "tokens": 5003, "experts": 160, "top_k": 6,
         "sequences": 7, "scoring": "softmax", "dtype": "bf16", "grad": True},
        # a training step of 16384 tokens, sigmoid scores
        {"name": "balance train", "op": "balance", "tokens": 16384, "experts": 256, "top_k": 8,
         "sequences": 0, "scoring": "sigmoid", "dtype": "fp32", "grad": True},
        # one token through a 4-bit projection
        {"name": "int4 decode", "op": "int4", "rows": 1, "cols": 4096, "depth": 7168, "group": 128,
         "zero": False, "bias": False, "dtype": "bf16"},
        # a batch of decode steps, odd output size, small groups with zero points, a bias
        {"name": "int4 ragged", "op": "int4", "rows": 37, "cols": 2047, "depth": 7168, "group": 32,
         "zero": True, "bias": True, "dtype": "fp16"},
        # a prefill batch through the same projection as the decode case
        {"name": "int4 prefill", "op": "int4", "rows": 8192, "cols": 4096, "depth": 7168,
         "group": 128, "zero": False, "bias": False, "dtype": "bf16"},
        # decode: 64 routed rows over the 32 experts of a rank, gate|up weights
        {"name": "int4 experts decode", "op": "experts", "rows": 64, "cols": 4096, "depth": 7168,
         "group": 128, "zero": False, "local": 32, "dtype": "bf16"},
        # prefill: 8192 routed rows over the same experts, down projection
        {"name": "int4 experts prefill", "op": "experts", "rows": 8192, "cols": 7168,
         "depth": 2048, "group": 64, "zero": True, "local": 32, "dtype": "bf16"},
        # a projection's weights put into 4 bits and read back for a check
        {"name": "int4 weights", "op": "weights", "local": 1, "cols": 4096, "depth": 7168,
         "group": 128, "zero": False, "dtype": "bf16"},
        # the weights of some experts, small groups with zero points, an odd number of channels
        {"name": "int4 weights experts", "op": "weights", "local": 8, "cols": 1407, "depth": 2048,
         "group": 32, "zero": True, "dtype": "fp16"},
        # one decode step of 16 sequences: the expert layer's input leaves as e4m3 with its scales
        {"name": "layer norm decode", "op": "norm", "tokens": 16, "hidden": 7168, "dtype": "bf16",
         "branch": True, "bias": True, "quantize": True, "grad": False},
        # a training step
        {"name": "layer norm train", "op": "norm", "tokens": 4096, "hidden": 7168, "dtype": "bf16",
         "branch": True, "bias": True, "quantize": False, "grad": True},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["balance", "int4", "experts", "weights", "norm", "norm"])
    if op == "balance":
        experts = rng.choice([8, 16, 64, 100, 128, 160, 256])
        return {"op": op, "tokens": _log(rng, 1, 16000), "experts": experts,
                "top_k": rng.choice([1, 2, 4, 6, 8]), "sequences": rng.choice([0, 0, 1, 5, 40]),
                "scoring": rng.choice(["softmax", "sigmoid"]),
                "dtype": rng.choice(["bf16", "fp16", "fp32"]), "grad": rng.random() < 0.7}
    if op == "weights":
        return {"op": op, "local": rng.choice([1, 1, 4, 8]), "cols": _log(rng, 64, 1800),
                "depth": 32 * _log(rng, 2, 100), "group": rng.choice([32, 64, 128]),
                "zero": rng.random() < 0.5, "dtype": rng.choice(["bf16", "fp16", "fp32"])}
    if op in ("int4", "experts"):
        case = {"op": op, "rows": _log(rng, 1, 6000), "cols": _log(rng, 64, 4000),
                "depth": 32 * _log(rng, 4, 220), "group": rng.choice([32, 64, 128, 128]),
                "zero": rng.random() < 0.5, "dtype": rng.choice(["bf16", "fp16"])}
        if op == "int4":
            case["bias"] = rng.random() < 0.5
        else:
            case["local"] = rng.choice([4, 8, 20, 32])
        return case
    quantize = rng.random() < 0.25
    return {"op": op, "tokens": _log(rng, 1, 4000),
            "hidden": 128 * _log(rng, 1, 56) if quantize else _log(rng, 64, 7100),
            "dtype": rng.choice(["bf16", "fp16", "fp32"]), "branch": rng.random() < 0.6,
            "bias": rng.random() < 0.7, "quantize": quantize,
            "grad": not quantize and rng.random() < 0.6}


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _groups(case):
    return -(-case["depth"] // case["group"])


def _prepare_balance(case, g, s):
    T, E, K = case["tokens"], case["experts"], min(case["top_k"], case["experts"])
    logits = _randn(g, T, E) + 0.7 * _randn(g, E)
    s["logits"] = logits.to(DTYPES[case["dtype"]]).requires_grad_(case["grad"])
    s["ids"] = s["logits"].detach().float().topk(K, dim=1).indices.to(torch.int32).contiguous()
    s["base"] = None
    if case["sequences"]:
        # ascending bases from row 0; the rows behind the last are padding
        cut = torch.rand(case["sequences"], generator=g, device="cuda").cumsum(0)
        cut = (cut / cut[-1] * (T - T // 20)).to(torch.int32)
        s["base"] = torch.cat([cut.new_zeros(1), cut])
    if case["grad"]:
        s["g"] = torch.rand((), generator=g, device="cuda") + 0.5


def _prepare_products(case, g, s):
    M, N, K, E = case["rows"], case["cols"], case["depth"], case.get("local", 1)
    dt = DTYPES[case["dtype"]]
    s["x"] = (_randn(g, M, K) * torch.exp(0.5 * _randn(g, M, 1))).to(dt)
    packed = torch.randint(0, 256, (E, N, K // 2), generator=g, device="cuda", dtype=torch.uint8)
    scale = ((torch.rand(E, N, _groups(case), generator=g, device="cuda") + 0.5) * 4e-3).to(dt)
    zero = None
    if case["zero"]:
        zero = torch.randint(5, 11, scale.shape, generator=g, device="cuda", dtype=torch.uint8)
    if case["op"] == "int4":
        s["packed"], s["scale"], s["zp"] = packed[0], scale[0], None if zero is None else zero[0]
        s["b"] = _randn(g, N) if case["bias"] else None
        return
    s["packed"], s["scale"], s["zp"] = packed, scale, zero
    popular = torch.softmax(0.7 * _randn(g, E), 0)
    ids = torch.multinomial(popular, M, replacement=True, generator=g)
    count = torch.bincount(ids, minlength=E)
    s["base"] = torch.cat([count.new_zeros(1), count.cumsum(0)]).to(torch.int32)
    s["most"] = int(count.max())


def _prepare_norm(case, g, s):
    T, H, grad, dt = case["tokens"], case["hidden"], case["grad"], DTYPES[case["dtype"]]
    # a residual stream of a few units that is not centred, a few channels far larger
    big = 1.0 + 20.0 * (torch.rand(H, generator=g, device="cuda") < 0.002)
    s["residual"] = (_randn(g, T, H) * 2 * big + 0.5).to(dt).requires_grad_(grad)
    if case["branch"]:
        s["x"] = _randn(g, T, H).to(dt).requires_grad_(grad)
    s["w"] = (1 + 0.1 * _randn(g, H)).to(dt).requires_grad_(grad)
    if case["bias"]:
        s["b"] = (0.1 * _randn(g, H)).to(dt).requires_grad_(grad)
    if grad:
        s["g_hidden"] = _randn(g, T, H).to(dt)
        s["g_normed"] = _randn(g, T, H).to(dt)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    s = {"case": dict(case)}
    if case["op"] == "balance":
        _prepare_balance(case, g, s)
    elif case["op"] in ("int4", "experts"):
        _prepare_products(case, g, s)
    elif case["op"] == "weights":
        shape = (case["local"], case["cols"], case["depth"])
        s["w"] = (0.02 * _randn(g, *shape)).to(DTYPES[case["dtype"]])
    else:
        _prepare_norm(case, g, s)
    return s


# ------------------------------------------------------------------ plain forms (32 bits)
def _plain_rows(base, T):
    """The sequence of every row, whether it has one, and the sequences' lengths."""
    row = torch.arange(T, device=base.device)
    seq = (row[:, None] >= base[None, 1:]).sum(1)
    live = (row >= base[0]) & (row < base[-1])
    return seq.clamp(max=base.numel() - 2), live, (base[1:] - base[:-1]).float()


def _plain_balance(s):
    case = s["case"]
    logits = s["logits"].detach().float().requires_grad_(case["grad"])
    T, E = logits.shape
    K = s["ids"].shape[1]
    base = s["base"]
    whole = base is None
    if whole:
        base = torch.zeros(2, dtype=torch.int32, device=logits.device)
        base[1:] += T
    base = base.long()
    S = base.numel() - 1
    seq, live, length = _plain_rows(base, T)
    ids = s["ids"].long()
    counted = live[:, None] & (ids >= 0) & (ids < E)
    at = torch.where(counted, seq[:, None] * E + ids, S * E).reshape(-1)
    counts = torch.zeros(S * E + 1, dtype=torch.long, device=logits.device)
    counts.scatter_add_(0, at, torch.ones_like(at))
    counts = counts[:S * E].view(S, E)
    if case["scoring"] == "softmax":
        e = torch.exp(logits - logits.detach().amax(1, keepdim=True))
    else:
        e = 1 / (1 + torch.exp(-logits))
    p = e / e.sum(1, keepdim=True)
    p = torch.where(live[:, None], p, 0.0)
    sums = torch.zeros(S, E, device=logits.device).index_add(0, seq, p)
    n = length.clamp(min=1)[:, None]
    each = ((counts.float() * (E / K) / n) * (sums / n)).sum(1)
    loss = torch.where(length > 0, each, 0.0).sum() / (length > 0).sum().clamp(min=1)
    got = {"loss": loss.detach(), "counts": (counts[0] if whole else counts).int()}
    if case["grad"]:
        got["d_logits"] = torch.autograd.grad(loss, logits, s["g"])[0].to(s["logits"].dtype)
    return got


def _plain_weights(packed, scale, zero, group):
    """The weights that 4-bit values, group scales and zero points stand for, in 32 bits."""
    K = packed.shape[-1] * 2
    q = torch.stack([packed & 15, packed >> 4], -1).reshape(*packed.shape[:-1], K).float()
    of = torch.arange(K, device=packed.device) // group
    z = 8.0 if zero is None else zero.float()[..., of]
    return (q - z) * scale.float()[..., of]


def _plain_int4(s):
    w = _plain_weights(s["packed"], s["scale"], s["zp"], s["case"]["group"])
    y = s["x"].float() @ w.t()
    if s["b"] is not None:
        y = y + s["b"]
    return {"y": y.to(s["x"].dtype)}


def _plain_experts(s):
    w = _plain_weights(s["packed"], s["scale"], s["zp"], s["case"]["group"])
    x, base = s["x"], s["base"].long()
    row = torch.arange(x.shape[0], device=x.device)
    at = base[:-1, None] + torch.arange(s["most"], device=x.device)
    acc = torch.bmm(x.float()[at.clamp(max=x.shape[0] - 1)], w.transpose(1, 2))
    e = (row[:, None] >= base[None, 1:]).sum(1)
    return {"y": acc[e, row - base[e]].to(x.dtype)}


def _least(w):
    """The smallest scale: one that its type can hold."""
    return 2.0 ** (-24 if w.dtype == torch.float16 else -100)


def _plain_quantise(s):
    w, case = s["w"], s["case"]
    E, N, K = w.shape
    G, n = case["group"], _groups(case)
    pad = torch.zeros(E, N, n * G, device=w.device)
    pad[:, :, :K] = w.float()
    blocks = pad.view(E, N, n, G)
    if case["zero"]:
        low, high = blocks.amin(3).clamp(max=0), blocks.amax(3).clamp(min=0)
        step = (high - low) / torch.full_like(high, 15)
    else:
        step = blocks.abs().amax(3) / torch.full_like(blocks[..., 0], 7)
    scale = step.clamp(min=_least(w)).to(w.dtype).float()
    if case["zero"]:
        zero = torch.round(-low / scale).clamp(0, 15)
        q = (torch.round(blocks / scale[..., None]) + zero[..., None]).clamp(0, 15)
    else:
        zero = torch.full_like(scale, 8)
        q = (torch.round(blocks / scale[..., None]) + 8).clamp(1, 15)
    back = (q - zero[..., None]) * scale[..., None]
    got = {"scale": scale.to(w.dtype), "back": back.view(E, N, n * G)[:, :, :K].to(w.dtype)}
    if case["zero"]:
        got["zero"] = zero.to(torch.uint8)
    return got


def _plain_norm(s):
    case, eps = s["case"], 1e-5
    names = [n for n in ("x", "residual", "w", "b") if n in s]
    v = {n: s[n].detach().float().requires_grad_(case["grad"]) for n in names}
    h = v["residual"] + v["x"] if case["branch"] else v["residual"]
    c = h - h.mean(1, keepdim=True)
    y = c * torch.rsqrt(c.square().mean(1, keepdim=True) + eps) * v["w"]
    if case["bias"]:
        y = y + v["b"]
    dt = s["residual"].dtype
    got = {"hidden": h.detach().to(dt)}
    if case["quantize"]:
        T, H = y.shape
        blocks = y.view(T, H // 128, 128)
        amax = blocks.abs().amax(2).clamp(min=1e-30)
        scale = amax / torch.full_like(amax, 448)
        got["q"] = (blocks / scale[:, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn).view(T, H)
        got["scale"] = scale.t().contiguous()
    else:
        got["normed"] = y.detach().to(dt)
    if case["grad"]:
        grads = torch.autograd.grad((h, y), [v[n] for n in names],
                                    (s["g_hidden"].float(), s["g_normed"].float()))
        got["grads"] = {n: d.to(dt) for n, d in zip(names, grads)}
    return got


# ------------------------------------------------------------------ the framework's calls
def _own_balance(s):
    import flashinfer_b200 as fb
    loss, counts = fb.balance_loss(s["logits"], s["ids"], scoring=s["case"]["scoring"],
                                   sequence_base=s["base"])
    got = {"loss": loss.detach(), "counts": counts}
    if s["case"]["grad"]:
        got["d_logits"] = torch.autograd.grad(loss, s["logits"], s["g"])[0]
    return got


def _own_int4(s):
    import flashinfer_b200 as fb
    return {"y": fb.int4_matmul(s["x"], s["packed"], s["scale"], s["zp"], s["b"],
                                group=s["case"]["group"])}


def _own_experts(s):
    import flashinfer_b200 as fb
    return {"y": fb.int4_expert_matmul(s["x"], s["packed"], s["scale"], s["base"], s["zp"],
                                       group=s["case"]["group"])}


def _own_quantise(s):
    import flashinfer_b200 as fb
    w, case = s["w"], s["case"]
    packed, scale, zero = fb.quantize_int4(w, group=case["group"], symmetric=not case["zero"])
    back = fb.dequantize_int4(packed, scale, zero, group=case["group"], out_dtype=w.dtype)
    got = {"scale": scale, "back": back}
    if case["zero"]:
        got["zero"] = zero
    return got


def _own_norm(s):
    import flashinfer_b200 as fb
    case = s["case"]
    h, y = fb.layer_norm(s.get("x"), s["residual"], weight=s["w"], bias=s.get("b"), eps=1e-5,
                         quantize=case["quantize"])
    if case["quantize"]:
        return {"hidden": h, "q": y[0], "scale": y[1]}
    got = {"hidden": h.detach(), "normed": y.detach()}
    if case["grad"]:
        names = [n for n in ("x", "residual", "w", "b") if n in s]
        grads = torch.autograd.grad((h, y), [s[n] for n in names], (s["g_hidden"], s["g_normed"]))
        got["grads"] = dict(zip(names, grads))
    return got


def run(state):
    op = state["case"]["op"]
    if own:
        return {"balance": _own_balance, "int4": _own_int4, "experts": _own_experts,
                "weights": _own_quantise, "norm": _own_norm}[op](state)
    return {"balance": _plain_balance, "int4": _plain_int4, "experts": _plain_experts,
            "weights": _plain_quantise, "norm": _plain_norm}[op](state)


def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["op"] == "balance":
        T, E, K, S = (case["tokens"], case["experts"], min(case["top_k"], case["experts"]),
                      max(1, case["sequences"]))
        b = size * T * E + 4 * (T * K + S * E + 1) + (4 * (S + 1) if case["sequences"] else 0)
        f = 8.0 * T * E
        if case["grad"]:  # the logits again, their gradient written
            b += 2 * size * T * E + 4
            f += 10.0 * T * E
        return {"bytes": b, "flops": f}
    if case["op"] in ("int4", "experts"):
        M, N, K, E = case["rows"], case["cols"], case["depth"], case.get("local", 1)
        used = min(E, M)
        b = size * M * (K + N) + used * N * (K // 2 + _groups(case) * (size + case["zero"]))
        b += 4 * N if case.get("bias") else 0
        b += 4 * (E + 1) if case["op"] == "experts" else 0
        return {"bytes": b, "flops": 2.0 * M * N * K}
    if case["op"] == "weights":
        rows = case["local"] * case["cols"]
        small = rows * (case["depth"] // 2 + _groups(case) * (size + case["zero"]))
        # weights read, 4-bit values written, read back and weights written
        return {"bytes": 2 * (size * rows * case["depth"] + small),
                "flops": 6.0 * rows * case["depth"]}
    T, H = case["tokens"], case["hidden"]
    n, params, ins = T * H, H * (1 + case["bias"]), 1 + case["branch"]
    b = size * ((ins + case["branch"]) * n + params)  # without a branch hidden is the residual
    b += n * (1 + 4 / 128) if case["quantize"] else size * n
    if case["grad"]:  # both gradients and the inputs read, every input's gradient written
        b += size * ((2 + ins) * n + params) + size * (n + params)
    return {"bytes": b, "flops": (30.0 if case["grad"] else 10.0) * n}


# ------------------------------------------------------------------ 64 bits, from the definitions
def _exact_balance(s):
    z = s["logits"].detach().double()
    T, E = z.shape
    K = s["ids"].shape[1]
    base = [0, T] if s["base"] is None else s["base"].tolist()
    if s["case"]["scoring"] == "softmax":
        p, slope = torch.softmax(z, 1), 1.0
    else:
        p, slope = torch.sigmoid(z), torch.sigmoid(-z)
        p = p / p.sum(1, keepdim=True)
    spans = [(a, b) for a, b in zip(base[:-1], base[1:]) if b > a]
    loss = torch.zeros((), dtype=torch.float64, device="cuda")
    grad = torch.zeros_like(z)
    for a, b in spans:
        picks = s["ids"][a:b].reshape(-1).long()
        count = torch.bincount(picks[(picks >= 0) & (picks < E)], minlength=E).double()
        factor = count * E / (K * (b - a) ** 2 * len(spans))
        loss = loss + (factor * p[a:b].sum(0)).sum()
        grad[a:b] = p[a:b] * (factor - (p[a:b] * factor).sum(1, keepdim=True))
    got = {"loss": loss, "counts": None}
    if s["case"]["grad"]:
        got["d_logits"] = grad * slope * s["g"].double()
    return got


def _exact_weights(packed, scale, zero, group):
    w = torch.empty(*packed.shape, 2, dtype=torch.float64, device=packed.device)
    w[..., 0], w[..., 1] = packed % 16, packed // 16
    w = w.flatten(-2)
    K = w.shape[-1]
    for k in range(0, K, group):
        at = (..., slice(k, min(k + group, K)))
        w[at] -= 8 if zero is None else zero[..., k // group, None].double()
        w[at] *= scale[..., k // group, None].double()
    return w


def _exact_products(s):
    x, group = s["x"].double(), s["case"]["group"]
    if s["case"]["op"] == "int4":
        y = torch.mm(x, _exact_weights(s["packed"], s["scale"], s["zp"], group).t())
        return {"y": y if s["b"] is None else y + s["b"].double()}
    base = s["base"].tolist()
    y = torch.zeros(x.shape[0], s["packed"].shape[1], dtype=torch.float64, device="cuda")
    for e, (lo, hi) in enumerate(zip(base[:-1], base[1:])):
        if lo < hi:
            zp = None if s["zp"] is None else s["zp"][e]
            y[lo:hi] = torch.mm(x[lo:hi], _exact_weights(s["packed"][e], s["scale"][e], zp,
                                                         group).t())
    return {"y": y}


def _exact_quantise(s):
    case, w = s["case"], s["w"].double()
    scale = []
    for k in range(0, w.shape[2], case["group"]):
        block = w[:, :, k:k + case["group"]]
        if case["zero"]:
            step = (block.amax(2).clamp(min=0) - block.amin(2).clamp(max=0)) / 15
        else:
            step = block.abs().amax(2) / 7
        scale.append(step.clamp(min=_least(s["w"])))
    # the values read back go by which side of a border a weight falls on, with the rounded scale
    got = {"scale": torch.stack(scale, 2), "back": None}
    if case["zero"]:
        got["zero"] = None
    return got


def _exact_norm(s):
    case, eps = s["case"], 1e-5
    h = s["residual"].detach().double()
    if case["branch"]:
        h = h + s["x"].detach().double()
    w = s["w"].detach().double()
    T, H = h.shape
    mean = h.sum(1, keepdim=True) / H
    r = 1 / torch.sqrt(((h - mean) ** 2).sum(1, keepdim=True) / H + eps)
    n = (h - mean) * r
    y = n * w
    if case["bias"]:
        y = y + s["b"].detach().double()
    got = {"hidden": h}
    if case["quantize"]:
        amax = y.view(T, H // 128, 128).abs().amax(2).clamp(min=1e-30)
        got["q"] = (y.view(T, H // 128, 128) / (amax / 448)[:, :, None]).view(T, H)
        got["scale"] = (amax / 448).t()
    else:
        got["normed"] = y
    if case["grad"]:
        dy = s["g_normed"].double()
        u = dy * w
        mean_u, mean_un = u.sum(1, keepdim=True) / H, (u * n).sum(1, keepdim=True) / H
        dh = s["g_hidden"].double() + r * (u - mean_u - n * mean_un)
        grads = {"x": dh} if case["branch"] else {}
        grads.update({"residual": dh, "w": (dy * n).sum(0)})
        if case["bias"]:
            grads["b"] = dy.sum(0)
        got["grads"] = grads
    return got


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"balance": _exact_balance, "int4": _exact_products, "experts": _exact_products,
                "weights": _exact_quantise, "norm": _exact_norm}[case["op"]](s)
