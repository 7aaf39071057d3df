"""Cases of three operators of a training step, each in a plain form and through the framework:

* ``rotary``        per-head RMS norm of queries and keys with the rotary embedding in the same
                    pass, or the rotary embedding alone (interleaved or half layout, the whole
                    head or its first lanes, frequencies scaled for long contexts)
* ``linear_ce``     cross entropy of a vocabulary projection that keeps no logits, with the
                    gradients of the hidden states and of the projection
* ``newton_schulz`` orthogonalised updates of a stack of weight matrices

``own`` chooses between the plain form (elementary torch operations in 32 bits, rounded once)
and the framework's calls.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
NORM_EPS = 1e-5
THETA = 10000.0
TRAINED = 4096           # positions a scaled table was trained on
IGNORE = -100
QUINTIC = (3.4445, -4.7750, 2.0315)
NS_STEPS = 5
NS_EPS = 1e-7


def listed():
    return [
        # one new token for each of 16 requests far into a long cache: grouped heads, latency
        dict(name="qk-decode", op="rotary", norm=True, backward=False, batch=16, tokens=1,
             heads=32, kv_heads=8, dim=128, rotated=128, layout="half", scaling="parts",
             table=131072, dtype="bf16"),
        # queries and keys of a microbatch of the 324M configuration, training
        dict(name="qk-train-324m", op="rotary", norm=True, backward=True, batch=4, tokens=1024,
             heads=16, kv_heads=16, dim=64, rotated=64, layout="interleaved", scaling="none",
             table=1024, dtype="bf16"),
        # a long-context training microbatch with grouped heads
        dict(name="qk-train-long", op="rotary", norm=True, backward=True, batch=2, tokens=32768,
             heads=32, kv_heads=8, dim=128, rotated=128, layout="half", scaling="parts",
             table=65536, dtype="bf16"),
        # rotation alone of the first lanes of each head, odd length, full precision
        dict(name="rotary-part-fp32", op="rotary", norm=False, backward=True, batch=3, tokens=2053,
             heads=12, kv_heads=12, dim=64, rotated=24, layout="half", scaling="linear",
             table=8192, dtype="fp32"),
        # scoring a short ragged batch against a large vocabulary: the loss of each token
        dict(name="ce-score", op="linear_ce", backward=False, tokens=173, dim=768, vocab=50257,
             ignored=0.3, dtype="fp16"),
        # the head of the 22M configuration
        dict(name="ce-train-22m", op="linear_ce", backward=True, tokens=1024, dim=512, vocab=10000,
             ignored=0.0, dtype="bf16"),
        # the head of the 324M configuration, one microbatch
        dict(name="ce-train-324m", op="linear_ce", backward=True, tokens=4096, dim=1024,
             vocab=10000, ignored=0.0, dtype="bf16"),
        # a large vocabulary, where the logits would not be kept
        dict(name="ce-train-large", op="linear_ce", backward=True, tokens=8192, dim=2048,
             vocab=131072, ignored=0.1, dtype="bf16"),
        # one small matrix
        dict(name="ns-one-small", op="newton_schulz", batch=1, rows=128, cols=384, dtype="fp32"),
        # an odd stack, as an adapter or a trimmed vocabulary gives
        dict(name="ns-odd", op="newton_schulz", batch=3, rows=1000, cols=337, dtype="bf16"),
        # attention projections of the 324M configuration: 4 of each of 24 layers
        dict(name="ns-attn-324m", op="newton_schulz", batch=96, rows=1024, cols=1024,
             dtype="fp32"),
        # gate and up projections of the 324M configuration: 2 of each of 24 layers, tall
        dict(name="ns-ffn-324m", op="newton_schulz", batch=48, rows=2752, cols=1024,
             dtype="fp32"),
    ]


def _spread(rng, low, high):
    """An integer whose logarithm is uniform over [low, high]."""
    return min(high, max(low, round(math.exp(rng.uniform(math.log(low), math.log(high))))))


def draw(rng):
    op = rng.choice(("rotary", "linear_ce", "newton_schulz"))
    if op == "rotary":
        tokens = _spread(rng, 1, 32768)
        dim = rng.choice((32, 64, 80, 96, 128, 192, 256))
        kv_heads = rng.choice((1, 2, 4, 8, 16))
        heads = kv_heads * rng.choice((1, 2, 4, 8) if kv_heads < 8 else (1, 2, 4))
        budget = 2 * 32768 * 40 * 128 // ((heads + kv_heads) * dim)
        tokens = min(tokens, budget)
        return dict(op=op, norm=rng.random() < 0.7, backward=rng.random() < 0.6,
                    batch=_spread(rng, 1, max(1, min(64, budget // tokens))), tokens=tokens,
                    heads=heads, kv_heads=kv_heads, dim=dim,
                    rotated=dim if rng.random() < 0.5 else 2 * rng.randint(1, dim // 2),
                    layout=rng.choice(("interleaved", "half")),
                    scaling=rng.choice(("none", "linear", "parts")),
                    table=_spread(rng, tokens, 131072), dtype=rng.choice(("bf16", "fp16", "fp32")))
    if op == "linear_ce":
        dim = 8 * _spread(rng, 8, 512)
        vocab = _spread(rng, 2, 131072)
        most = 8192 * 2048 * 131072 // (dim * vocab)
        return dict(op=op, backward=rng.random() < 0.7, tokens=_spread(rng, 1, min(16384, most)),
                    dim=dim, vocab=vocab, ignored=rng.choice((0.0, 0.1, 0.5)),
                    dtype=rng.choice(("bf16", "fp16")))
    rows, cols = _spread(rng, 16, 4096), _spread(rng, 16, 4096)
    one = _ns_flops(1, rows, cols)
    return dict(op=op, batch=_spread(rng, 1, max(1, min(96, int(_ns_flops(48, 2752, 1024) / one)))),
                rows=rows, cols=cols, dtype=rng.choice(("fp32", "bf16")))


# ------------------------------------------------------------------------- inputs --
def _inverse_frequencies(case):
    """Angle per position of each rotated pair, in 64 bits on the host.

    "linear" divides every frequency by 4; "parts" divides by 8 the frequencies that turn at
    most once within the positions trained on, keeps those that turn at least 4 times, and
    interpolates in between.
    """
    rotated = case["rotated"]
    freq = THETA ** (-torch.arange(0, rotated, 2, dtype=torch.float64) / rotated)
    if case["scaling"] == "linear":
        return freq / 4.0
    if case["scaling"] == "parts":
        turns = TRAINED * freq / (2 * math.pi)
        keep = ((turns - 1.0) / 3.0).clamp(0.0, 1.0)
        return freq * keep + freq / 8.0 * (1.0 - keep)
    return freq


def prepare(case, seed):
    dev = torch.device("cuda", torch.cuda.current_device())
    gen = torch.Generator(device=dev).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def randn(*shape, scale=1.0):
        return torch.randn(*shape, device=dev, generator=gen) * scale

    state = {"case": dict(case)}
    if case["op"] == "rotary":
        B, T, H, G, D = (case[k] for k in ("batch", "tokens", "heads", "kv_heads", "dim"))
        # one packed projection [B, T, q | k | v heads, D], as the model's matrix product leaves it
        packed = randn(B, T, H + 2 * G, D).to(dtype)
        state["q"] = packed[:, :, :H].permute(0, 2, 1, 3)
        state["k"] = packed[:, :, H:H + G].permute(0, 2, 1, 3)
        first = torch.randint(0, case["table"] - T + 1, (B, 1), device=dev, generator=gen)
        state["positions"] = first + torch.arange(T, device=dev)
        freq = _inverse_frequencies(case)
        angles = torch.arange(case["table"], dtype=torch.float64, device=dev)[:, None] * freq.to(dev)
        state["cos"], state["sin"] = angles.cos().float(), angles.sin().float()
        state["freq"] = freq.to(dev)
        if case["norm"]:
            state["q_weight"] = 1.0 + randn(D, scale=0.2)
            state["k_weight"] = 1.0 + randn(D, scale=0.2)
        if case["backward"]:
            # attention's gradients arrive token-major
            state["dq"] = randn(B, T, H, D).to(dtype).permute(0, 2, 1, 3)
            state["dk"] = randn(B, T, G, D).to(dtype).permute(0, 2, 1, 3)
    elif case["op"] == "linear_ce":
        N, D, V = case["tokens"], case["dim"], case["vocab"]
        state["weight"] = randn(V, D, scale=1.2 / D ** 0.5).to(dtype)
        targets = torch.randint(0, V, (N,), device=dev, generator=gen)
        # normalised hidden states that already lean towards their target, as in a trained model
        lean = state["weight"][targets].float() * randn(N, 1).abs() * 3.0
        hidden = randn(N, D) + lean
        hidden = hidden * torch.rsqrt(hidden.square().mean(-1, keepdim=True) + NORM_EPS)
        state["hidden"] = hidden.to(dtype)
        dropped = torch.rand(N, device=dev, generator=gen) < case["ignored"]
        dropped[0] = False
        state["targets"] = targets.masked_fill(dropped, IGNORE)
    else:
        L, m, n = case["batch"], case["rows"], case["cols"]
        rank = max(1, min(m, n) // 4)
        # gradients of linear layers: a decaying low-rank part and noise
        falling = torch.exp(-3.0 * torch.arange(rank, device=dev) / rank)
        update = torch.bmm(randn(L, m, rank) * falling, randn(L, rank, n)) / rank ** 0.5
        state["update"] = ((update + 0.2 * randn(L, m, n)) * 1e-3).to(dtype)
    return state


# -------------------------------------------------------------------------- calls --
def run(state):
    case = state["case"]
    if case["op"] == "rotary":
        return _own_rotary(state) if own else _plain_rotary(state)
    if case["op"] == "linear_ce":
        return _own_linear_ce(state) if own else _plain_linear_ce(state)
    if own:
        from systems_for_llms_b200.ops.newton_schulz import newton_schulz
        return newton_schulz(state["update"], steps=NS_STEPS, coefficients=QUINTIC, eps=NS_EPS)
    return _plain_newton_schulz(state["update"])


def _own_rotary(state):
    from systems_for_llms_b200.ops.rotary import qk_norm_rotary, rotary
    case = state["case"]
    names = ["q", "k"] + (["q_weight", "k_weight"] if case["norm"] else [])
    leaves = [state[name].detach().requires_grad_(case["backward"]) for name in names]
    tables = (state["cos"], state["sin"], state["positions"])
    if case["norm"]:
        outs = qk_norm_rotary(*leaves, *tables, eps=NORM_EPS, layout=case["layout"])
    else:
        outs = tuple(rotary(x, *tables, layout=case["layout"]) for x in leaves)
    if not case["backward"]:
        return outs
    grads = torch.autograd.grad(outs, leaves, (state["dq"], state["dk"]))
    return tuple(x.detach() for x in outs) + grads


def _own_linear_ce(state):
    from systems_for_llms_b200.ops.linear_loss import linear_cross_entropy
    backward = state["case"]["backward"]
    leaves = [state[name].detach().requires_grad_(backward) for name in ("hidden", "weight")]
    loss = linear_cross_entropy(*leaves, state["targets"], ignore_index=IGNORE,
                                reduction="mean" if backward else "none")
    if not backward:
        return loss
    return (loss.detach(),) + torch.autograd.grad(loss, leaves)


# -------------------------------------------------------------------- plain forms --
def _pairs(x, layout):
    """The two lanes of each rotated pair."""
    return (x[..., 0::2], x[..., 1::2]) if layout == "interleaved" else x.chunk(2, dim=-1)


def _join(a, b, layout):
    if layout == "interleaved":
        return torch.stack((a, b), dim=-1).flatten(-2)
    return torch.cat((a, b), dim=-1)


def _turn(x, cos, sin, rotated, layout):
    a, b = _pairs(x[..., :rotated], layout)
    return torch.cat((_join(a * cos - b * sin, a * sin + b * cos, layout), x[..., rotated:]), dim=-1)


def _plain_one(x, weight, grad, cos, sin, rotated, layout):
    """Norm and rotation of one tensor, and what its gradient turns into."""
    wide = x.float()
    if weight is not None:
        rstd = torch.rsqrt(wide.square().mean(-1, keepdim=True) + NORM_EPS)
        unit = wide * rstd
        out = _turn(unit * weight, cos, sin, rotated, layout)
    else:
        out = _turn(wide, cos, sin, rotated, layout)
    if grad is None:
        return out.to(x.dtype), None, None
    back = _turn(grad.float(), cos, -sin, rotated, layout)
    if weight is None:
        return out.to(x.dtype), back.to(x.dtype), None
    d_weight = (back * unit).sum(dim=(0, 1, 2))
    d_unit = back * weight
    dx = rstd * (d_unit - unit * (d_unit * unit).mean(-1, keepdim=True))
    return out.to(x.dtype), dx.to(x.dtype), d_weight


def _plain_rotary(state):
    case = state["case"]
    angles = (state["positions"].double()[:, None, :, None] * state["freq"])
    cos, sin = angles.cos().float(), angles.sin().float()
    common = (cos, sin, case["rotated"], case["layout"])
    q, dq, dqw = _plain_one(state["q"], state.get("q_weight"), state.get("dq"), *common)
    k, dk, dkw = _plain_one(state["k"], state.get("k_weight"), state.get("dk"), *common)
    if not case["backward"]:
        return q, k
    return (q, k, dq, dk, dqw, dkw) if case["norm"] else (q, k, dq, dk)


def _plain_linear_ce(state):
    hidden, weight, targets = state["hidden"].float(), state["weight"].float(), state["targets"]
    valid = targets != IGNORE
    count = valid.sum()
    index = torch.where(valid, targets, 0)[:, None]
    logits = hidden @ weight.t()
    logits = logits - logits.amax(dim=-1, keepdim=True)
    picked = logits.gather(-1, index)
    p = logits.exp_()
    total = p.sum(dim=-1, keepdim=True)
    loss = torch.where(valid, (total.log() - picked)[:, 0], 0.0)
    if not state["case"]["backward"]:
        return loss
    loss = loss.sum() / count
    p /= total
    p.scatter_add_(-1, index, torch.full_like(picked, -1.0))
    p *= (valid / count)[:, None]
    return loss, (p @ weight).to(state["hidden"].dtype), (p.t() @ hidden).to(state["weight"].dtype)


def _plain_newton_schulz(update):
    a, b, c = QUINTIC
    x = update.float()
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + NS_EPS)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for _ in range(NS_STEPS):
        gram = x @ x.mT
        x = a * x + (b * gram + c * (gram @ gram)) @ x
    return (x.mT if tall else x).contiguous().to(torch.bfloat16)


# --------------------------------------------------------------------------- work --
def _ns_flops(batch, rows, cols):
    """The two Gram-sized products are symmetric: half of each is enough."""
    m, n = min(rows, cols), max(rows, cols)
    return float(batch * NS_STEPS * (m * m * n + m * m * m + 2 * m * m * n))


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}[case["dtype"]]
    if case["op"] == "rotary":
        rows = case["batch"] * case["tokens"] * (case["heads"] + case["kv_heads"])
        tensor = rows * case["dim"] * size
        pairs = min(case["table"], case["batch"] * case["tokens"]) * case["rotated"] // 2
        # x and y forward; with a gradient also dy and dx (x is still needed by the norm alone)
        moved = 2 * tensor + pairs * 8 + case["batch"] * case["tokens"] * 8
        flops = rows * (case["rotated"] * 3 + (case["dim"] * 4 if case["norm"] else 0))
        if case["backward"]:
            moved += 2 * tensor + (case["dim"] * 16 if case["norm"] else 0)
            flops += rows * (case["rotated"] * 3 + (case["dim"] * 10 if case["norm"] else 0))
        return {"bytes": float(moved), "flops": float(flops)}
    if case["op"] == "linear_ce":
        N, D, V = case["tokens"], case["dim"], case["vocab"]
        operands = (N * D + V * D) * size
        times = 2 if case["backward"] else 1
        return {"bytes": float(operands * times + N * 8 + (4 if case["backward"] else 4 * N)),
                "flops": float(N) * D * V * (6 if case["backward"] else 2)}
    L, m, n = case["batch"], case["rows"], case["cols"]
    return {"bytes": float(L * m * n * (size + 2)), "flops": _ns_flops(L, m, n)}


# -------------------------------------------------------------------------- exact --
def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, state)
    if case["op"] == "linear_ce":
        return _exact_linear_ce(case, state)
    # X p(X^T X) by Horner's rule on the left Gram matrix, one matrix of the stack at a time
    a, b, c = QUINTIC
    out = []
    for one in state["update"]:
        x = one.double()
        x = x / (torch.linalg.matrix_norm(x) + NS_EPS)
        for _ in range(NS_STEPS):
            if x.shape[0] <= x.shape[1]:
                gram = x @ x.t()
                x = a * x + gram @ (b * x + c * (gram @ x))
            else:
                gram = x.t() @ x
                x = a * x + (b * x + c * (x @ gram)) @ gram
        out.append(x)
    return torch.stack(out)


def _exact_rotary(case, state):
    """Each pair as a complex number, turned by a unit number; gradients by autograd."""
    lanes = torch.arange(case["rotated"], device=state["q"].device)
    if case["layout"] == "interleaved":
        first, second = lanes[0::2], lanes[1::2]
    else:
        first, second = lanes.chunk(2)
    angle = state["positions"].double()[:, None, :, None] * state["freq"]
    unit = torch.polar(torch.ones_like(angle), angle)

    def form(x, weight):
        if weight is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / case["dim"] + NORM_EPS).sqrt() * weight
        turned = torch.complex(x[..., first], x[..., second]) * unit
        y = x.clone()
        y[..., first], y[..., second] = turned.real, turned.imag
        return y

    outs, grads, weights = [], [], []
    for name in ("q", "k"):
        x = state[name].double().requires_grad_(case["backward"])
        leaves = [x]
        if case["norm"]:
            leaves.append(state[name + "_weight"].double().requires_grad_(case["backward"]))
        y = form(x, leaves[1] if case["norm"] else None)
        outs.append(y.detach())
        if case["backward"]:
            got = torch.autograd.grad(y, leaves, state["d" + name].double())
            grads.append(got[0])
            weights += got[1:]
    return tuple(outs + grads + weights)


def _exact_linear_ce(case, state):
    """Strips of rows in 64 bits."""
    hidden, weight = state["hidden"].double(), state["weight"].double()
    targets = state["targets"]
    valid = targets >= 0
    count = int(valid.sum())
    strip = max(1, (1 << 28) // case["vocab"])
    losses = torch.zeros(case["tokens"], dtype=torch.float64, device=hidden.device)
    d_hidden, d_weight = torch.zeros_like(hidden), torch.zeros_like(weight)
    for begin in range(0, case["tokens"], strip):
        rows = slice(begin, begin + strip)
        keep = valid[rows].nonzero()[:, 0]
        if keep.numel() == 0:
            continue
        h, t = hidden[rows][keep], targets[rows][keep]
        logp = torch.log_softmax(h @ weight.t(), dim=-1)
        order = torch.arange(keep.numel(), device=h.device)
        losses[begin + keep] = -logp[order, t]
        if case["backward"]:
            g = logp.exp_()
            g[order, t] -= 1.0
            g /= count
            d_hidden[begin + keep] = g @ weight
            d_weight += g.t() @ h
    return (losses.sum() / count, d_hidden, d_weight) if case["backward"] else losses
