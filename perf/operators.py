"""The operators of an attention layer with rotary positions, and the cases they are measured on.

Three operators of ``tynx_b200.nn``: the rotary position embedding, the per-head
norm of queries and keys with the rotation in the same pass, and differential
attention, the difference of two softmax maps with a learned weight per head.
``run`` computes a case in plain torch operations, or, with ``own`` set, through
the framework.  Tensors are float32 (the framework's floating type), positions
and key lengths int64.

Layouts: heads are ``[batch, tokens, heads, head_dim]``.  Differential attention
takes two maps a head, ``q [batch, tokens, 2 * heads, d]`` and
``k [batch, keys, 2 * kv_heads, d]`` with the maps of head ``h`` at ``2 h`` and
``2 h + 1``, ``v [batch, keys, kv_heads, dv]`` and ``lam [heads]``; query heads
``h`` share key head ``h // (heads // kv_heads)``.
"""

import math

import torch

own = False

DEVICE = "cuda"
EPS = 1e-6


def listed():
    return [
        # the next token of eight sequences far into a long context, the frequencies blended
        # for a context of eight times the length they were trained on
        {"name": "rotary, one token, long context", "op": "rotary", "batch": 8, "tokens": 1, "heads": 32, "dim": 128,
         "rot": 128, "interleaved": False, "scaling": "yarn", "factor": 8.0, "start": 30011, "train": False},
        # a training batch, neighbouring elements rotate together
        {"name": "rotary, training, interleaved", "op": "rotary", "batch": 8, "tokens": 2048, "heads": 16, "dim": 64,
         "rot": 64, "interleaved": True, "scaling": "none", "factor": 1.0, "start": 0, "train": True},
        # a quarter of each head rotates, odd numbers of tokens and heads
        {"name": "rotary, part of the head, odd", "op": "rotary", "batch": 3, "tokens": 777, "heads": 5, "dim": 80,
         "rot": 20, "interleaved": False, "scaling": "linear", "factor": 4.0, "start": 5, "train": True},
        # one token of sixteen sequences, four query heads a key head
        {"name": "qk norm, one token", "op": "qk_norm", "batch": 16, "tokens": 1, "heads": 16, "kv_heads": 4, "dim": 128,
         "rot": 128, "interleaved": False, "scaling": "none", "factor": 1.0, "start": 4095, "train": False},
        # a training batch of long sequences
        {"name": "qk norm, training", "op": "qk_norm", "batch": 4, "tokens": 4096, "heads": 16, "kv_heads": 4, "dim": 128,
         "rot": 128, "interleaved": False, "scaling": "none", "factor": 1.0, "start": 0, "train": True},
        # two thirds of an odd head size rotate in neighbouring pairs
        {"name": "qk norm, training, odd", "op": "qk_norm", "batch": 5, "tokens": 333, "heads": 6, "kv_heads": 3, "dim": 96,
         "rot": 64, "interleaved": True, "scaling": "linear", "factor": 2.0, "start": 0, "train": True},
        # one token of eight sequences against their keys so far, which end at different lengths
        {"name": "diff, one token, long keys", "op": "diff", "batch": 8, "tokens": 1, "keys": 8190, "heads": 8,
         "kv_heads": 2, "d": 64, "dv": 128, "causal": False, "start": 0, "ragged": True, "train": False},
        # the token classifier's batch and width (256 sequences of 128 tokens, width 256) as two differential heads
        {"name": "diff, training, short sequences", "op": "diff", "batch": 256, "tokens": 128, "keys": 128, "heads": 2,
         "kv_heads": 2, "d": 64, "dv": 128, "causal": False, "start": 0, "ragged": False, "train": True},
        # a language model's training batch
        {"name": "diff, training, causal", "op": "diff", "batch": 2, "tokens": 2048, "keys": 2048, "heads": 8,
         "kv_heads": 4, "d": 64, "dv": 128, "causal": True, "start": 0, "ragged": False, "train": True},
        # odd sizes, padded sequences (one of them empty), three query heads to one key head
        {"name": "diff, training, odd and padded", "op": "diff", "batch": 5, "tokens": 413, "keys": 413, "heads": 3,
         "kv_heads": 1, "d": 40, "dv": 72, "causal": True, "start": 0, "ragged": True, "train": True},
        # sixty-four new tokens behind a context of 4032
        {"name": "diff, chunk behind a context", "op": "diff", "batch": 4, "tokens": 64, "keys": 4096, "heads": 8,
         "kv_heads": 4, "d": 64, "dv": 128, "causal": True, "start": 4032, "ragged": False, "train": False},
        # a long prompt
        {"name": "diff, long prompt", "op": "diff", "batch": 1, "tokens": 8192, "keys": 8192, "heads": 8,
         "kv_heads": 8, "d": 64, "dv": 128, "causal": True, "start": 0, "ragged": False, "train": False},
    ]


def _log(rng, low, high):
    """A whole number of [low, high], spread over its logarithm."""
    return min(high, int(math.exp(rng.uniform(math.log(low), math.log(high + 1)))))


def draw(rng):
    op = rng.choice(["rotary", "qk_norm", "diff"])
    if op == "diff":
        kv = rng.choice([1, 2, 3, 4, 8])
        heads = kv * rng.choice([1, 1, 2, 3])
        d = rng.choice([8, 24, 32, 40, 48, 64, 64, 64])
        dv = rng.choice([d, 2 * d, 2 * d, 72])
        if rng.random() < 0.25:  # one token, or a few, against many keys
            tokens, keys = rng.choice([1, 1, 2, 5]), _log(rng, 2, 16384)
            return {"op": op, "batch": rng.randint(1, 8), "tokens": tokens, "keys": max(keys, tokens), "heads": heads,
                    "kv_heads": kv, "d": d, "dv": dv, "causal": False, "start": 0, "ragged": rng.random() < 0.5,
                    "train": False}
        start = rng.choice([0, 0, _log(rng, 1, 1000)])
        tokens = min(_log(rng, 2, 3000), int(math.sqrt(7e7 / heads + start * start / 4) - start / 2))
        most = max(1, int(7e7 / (heads * tokens * (tokens + start))))
        return {"op": op, "batch": rng.randint(1, min(64, most)), "tokens": tokens, "keys": tokens + start,
                "heads": heads, "kv_heads": kv, "d": d, "dv": dv, "causal": rng.random() < 0.7, "start": start,
                "ragged": rng.random() < 0.3, "train": rng.random() < 0.7}
    dim = rng.choice([16, 40, 64, 64, 80, 96, 128, 128, 256])
    rot = rng.choice([dim, dim, dim // 2 // 2 * 2])
    heads = rng.randint(1, 32)
    kv = rng.choice([h for h in (1, 2, 3, 4, 8) if heads % h == 0]) if op == "qk_norm" else 0
    most = 16384 * 20 * 128 // ((heads + kv) * dim)
    tokens = rng.choice([1, _log(rng, 1, min(8192, most))])
    scaling = rng.choice(["none", "linear", "yarn"])
    case = {"op": op, "batch": _log(rng, 1, max(1, min(64, most // tokens))), "tokens": tokens, "heads": heads,
            "dim": dim, "rot": rot, "interleaved": rng.random() < 0.5, "scaling": scaling,
            "factor": 1.0 if scaling == "none" else rng.choice([2.0, 4.0, 8.0]), "start": rng.choice([0, _log(rng, 1, 100000)]),
            "train": tokens > 1 and rng.random() < 0.7}
    if op == "qk_norm":
        case["kv_heads"] = kv
    return case


ORIGINAL_LENGTH = 4096  # the context length that the blended frequencies start from


def _scaling(case):
    """The scaling argument of ``tynx_b200.nn.Rotary`` for a case."""
    if case["scaling"] == "none":
        return None
    if case["scaling"] == "linear":
        return {"type": "linear", "factor": case["factor"]}
    return {"type": "yarn", "factor": case["factor"], "original_length": ORIGINAL_LENGTH}


def _lengths(case):
    """The valid keys of each sequence: from none and one up to all of them."""
    b, s = case["batch"], case["keys"]
    if not case["ragged"]:
        return [s] * b
    if case["tokens"] <= 8:  # sequences being continued
        return [max(1, s - (i * s) // (2 * b)) for i in range(b)]
    return [0 if i == 0 and b > 1 else 1 if i == 1 and b > 2 else max(1, ((i + 1) * s) // b) for i in range(b)]


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE)
    gen.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    b, t = case["batch"], case["tokens"]
    state = {"case": case, "handles": {}}
    if case["op"] == "diff":
        s, h, hk, d, dv = case["keys"], case["heads"], case["kv_heads"], case["d"], case["dv"]
        state["q"] = normal(b, t, 2 * h, d)
        state["k"] = normal(b, s, 2 * hk, d)
        state["v"] = normal(b, s, hk, dv)
        state["lam"] = 0.2 + 0.6 * torch.rand(h, generator=gen, device=DEVICE)
        state["lengths"] = torch.tensor(_lengths(case), device=DEVICE) if case["ragged"] else None
        if case["train"]:
            state["dout"] = normal(b, t, h, dv)
        return state
    state["positions"] = (case["start"] + torch.arange(t, device=DEVICE))[None, :] + 3 * torch.arange(b, device=DEVICE)[:, None]
    if case["op"] == "rotary":
        state["x"] = normal(b, t, case["heads"], case["dim"])
        if case["train"]:
            state["dy"] = normal(b, t, case["heads"], case["dim"])
        return state
    for name, heads in (("q", case["heads"]), ("k", case["kv_heads"])):
        state[name] = normal(b, t, heads, case["dim"])
        state[name + "_weight"] = 1.0 + 0.1 * normal(case["dim"])
        if case["train"]:
            state["d" + name] = normal(b, t, heads, case["dim"])
    return state


# ---- the plain forms ---------------------------------------------------------


def _frequencies(case):
    """(radians a position of each rotating pair in 64 bits, the factor on cosine and sine)."""
    rot = case["rot"]
    i = torch.arange(0, rot, 2, dtype=torch.float64, device=DEVICE)
    base = 10000.0
    inv = base ** (-i / rot)
    if case["scaling"] == "linear":
        return inv / case["factor"], 1.0
    if case["scaling"] == "yarn":
        # pairs that turn more than 32 times over the original length keep their frequency, those
        # that turn less than once have it divided, the ones between are blended
        def pair(turns):
            return rot * math.log(ORIGINAL_LENGTH / (turns * 2 * math.pi)) / (2 * math.log(base))

        low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), rot - 1)
        ramp = ((i / 2 - low) / max(high - low, 0.001)).clamp(0, 1)
        return inv * (1 - ramp) + inv / case["factor"] * ramp, 0.1 * math.log(case["factor"]) + 1.0
    return inv, 1.0


def _angles(state):
    inv, factor = _frequencies(state["case"])
    angle = state["positions"].double()[..., None] * inv
    return (angle.cos() * factor).float()[:, :, None, :], (angle.sin() * factor).float()[:, :, None, :]


def _rotate(x, cos, sin, case):
    rot = case["rot"]
    if case["interleaved"]:
        a, b = x[..., 0:rot:2], x[..., 1:rot:2]
        turned = torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)
    else:
        a, b = x[..., : rot // 2], x[..., rot // 2 : rot]
        turned = torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    return torch.cat((turned, x[..., rot:]), -1)


def _plain_rotary(state):
    case = state["case"]
    cos, sin = _angles(state)
    y = _rotate(state["x"], cos, sin, case)
    return [y, _rotate(state["dy"], cos, -sin, case)] if case["train"] else [y]


def _plain_qk_norm(state):
    case = state["case"]
    cos, sin = _angles(state)

    def one(x, weight, dy):
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        unit = x * r
        y = _rotate(unit * weight, cos, sin, case)
        if dy is None:
            return y, None, None
        g = _rotate(dy, cos, -sin, case)
        gw = g * weight
        dx = r * (gw - unit * (gw * unit).mean(-1, keepdim=True))
        return y, dx, (g * unit).sum((0, 1, 2))

    yq, dq, dwq = one(state["q"], state["q_weight"], state.get("dq"))
    yk, dk, dwk = one(state["k"], state["k_weight"], state.get("dk"))
    return [yq, yk, dq, dk, dwq, dwk] if case["train"] else [yq, yk]


def _allowed(state):
    """[batch, tokens, keys]: whether a query sees a key."""
    case = state["case"]
    key = torch.arange(case["keys"], device=DEVICE)[None, None, :]
    ok = torch.ones(case["batch"], case["tokens"], case["keys"], dtype=torch.bool, device=DEVICE)
    if case["causal"]:
        ok = ok & (key <= torch.arange(case["tokens"], device=DEVICE)[None, :, None] + case["start"])
    if state["lengths"] is not None:
        ok = ok & (key < state["lengths"][:, None, None])
    return ok


def _plain_diff(state):
    case = state["case"]
    b, t, s, h, hk, d, dv = (case[n] for n in ("batch", "tokens", "keys", "heads", "kv_heads", "d", "dv"))
    g, scale = h // hk, d ** -0.5
    q = state["q"].view(b, t, hk, g, 2, d).permute(0, 2, 3, 4, 1, 5)
    k = state["k"].view(b, s, hk, 1, 2, d).permute(0, 2, 3, 4, 1, 5)
    v = state["v"].view(b, s, hk, 1, dv).permute(0, 2, 3, 1, 4)
    lam = state["lam"].view(1, hk, g, 1, 1)
    ok = _allowed(state)[:, None, None, None]
    score = (q @ k.transpose(-1, -2) * scale).masked_fill(~ok, float("-inf"))
    top = score.amax(-1, keepdim=True)
    p = torch.exp(score - top.masked_fill(top == float("-inf"), 0.0))
    a = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    w = a[:, :, :, 0] - lam * a[:, :, :, 1]
    out = (w @ v).permute(0, 3, 1, 2, 4).reshape(b, t, h, dv)
    if not case["train"]:
        return [out]
    dout = state["dout"].view(b, t, hk, g, dv).permute(0, 2, 3, 1, 4)
    dw = dout @ v.transpose(-1, -2)
    dvalue = (w.transpose(-1, -2) @ dout).sum(2).permute(0, 2, 1, 3)
    dlam = -(dw * a[:, :, :, 1]).sum((0, 3, 4)).reshape(h)
    da = torch.stack((dw, -lam * dw), 3)
    ds = a * (da - (a * da).sum(-1, keepdim=True)) * scale
    dq = (ds @ k).permute(0, 4, 1, 2, 3, 5).reshape(b, t, 2 * h, d)
    dk = (ds.transpose(-1, -2) @ q).sum(2).permute(0, 3, 1, 2, 4).reshape(b, s, 2 * hk, d)
    return [out, dq, dk, dvalue.contiguous(), dlam]


# ---- the framework's calls ---------------------------------------------------


def _tensors(state):
    """The state's buffers as the framework's tensors, as a program that trains or serves holds them."""
    import tynx_b200 as tx

    held = state["handles"]
    if not held:
        case = state["case"]
        for name, value in state.items():
            if isinstance(value, torch.Tensor):
                held[name] = tx.from_dlpack(value)
        if case["op"] != "diff":
            held["rotary"] = tx.nn.Rotary(case["rot"], interleaved=case["interleaved"], scaling=_scaling(case))
        if case["train"]:
            for name in ("x", "q", "k", "q_weight", "k_weight", "v", "lam"):
                if name in held:
                    held[name].requires_grad_()
    return held


def _run_own(state):
    import tynx_b200 as tx

    case, held = state["case"], _tensors(state)
    functional = tx.nn.functional
    if case["op"] == "rotary":
        outputs = [functional.rotary_embedding(held["x"], held["rotary"], held["positions"])]
        leaves, seeds = ("x",), ("dy",)
    elif case["op"] == "qk_norm":
        outputs = list(functional.qk_norm_rotary(held["q"], held["k"], held["q_weight"], held["k_weight"],
                                                 held["rotary"], held["positions"], eps=EPS))
        leaves, seeds = ("q", "k", "q_weight", "k_weight"), ("dq", "dk")
    else:
        outputs = [functional.differential_attention(held["q"], held["k"], held["v"], held["lam"], causal=case["causal"],
                                                     query_start=case["start"], key_lengths=held.get("lengths"))]
        leaves, seeds = ("q", "k", "v", "lam"), ("dout",)
    if case["train"]:
        tx.backward(outputs, [held[name] for name in seeds])
        for name in leaves:
            outputs.append(held[name].grad)
            held[name].grad = None
    return [torch.from_dlpack(t.detach()) for t in outputs]


def run(state):
    if own:
        return _run_own(state)
    return {"rotary": _plain_rotary, "qk_norm": _plain_qk_norm, "diff": _plain_diff}[state["case"]["op"]](state)


# ---- what a pass cannot do without -------------------------------------------


def _pairs(case):
    """Query-key pairs that some query sees, over the batch, for one head."""
    total = 0
    for n in _lengths(case):
        if not case["causal"]:
            total += case["tokens"] * n
        else:
            # query i sees min(n, i + start + 1) keys
            full = max(0, min(case["tokens"], case["tokens"] + case["start"] - n + 1))
            part = case["tokens"] - full
            total += full * n + part * (case["start"] + 1) + part * (part - 1) // 2
    return total


def work(case):
    b, t = case["batch"], case["tokens"]
    if case["op"] == "diff":
        h, hk, d, dv = case["heads"], case["kv_heads"], case["d"], case["dv"]
        seen = sum(min(n, t + case["start"]) if case["causal"] else n for n in _lengths(case))
        queries, values = b * t * 2 * h * d, b * t * h * dv
        keys = seen * hk * (2 * d + dv)
        pairs = _pairs(case) * h
        if not case["train"]:
            return {"bytes": 4 * (queries + keys + values), "flops": pairs * (4 * d + 2 * dv)}
        written = b * case["keys"] * hk * (2 * d + dv)
        return {"bytes": 4 * (2 * queries + keys + written + 2 * values), "flops": pairs * (4 * d + 2 * dv + 8 * d + 4 * dv)}
    rows = b * t * (case["heads"] + case.get("kv_heads", 0))
    values = rows * case["dim"]
    turned = rows * case["rot"]
    if case["op"] == "rotary":
        moved = 4 if case["train"] else 2
        return {"bytes": 4 * moved * values + 8 * b * t, "flops": 3 * turned * moved // 2}
    moved = 4 if case["train"] else 2  # x and the output's gradient in, y and the input's gradient out
    return {"bytes": 4 * moved * values + 8 * b * t, "flops": (3 * turned + 5 * values) * moved // 2}


# ---- the definitions in 64 bits ----------------------------------------------


def _exact_turn(x, state):
    """The rotation as a product of complex numbers, x in 64 bits."""
    case = state["case"]
    rot, n = case["rot"], case["rot"] // 2
    inv, factor = _frequencies(case)
    angle = state["positions"].to(torch.float64).unsqueeze(-1).mul(inv).unsqueeze(2)
    spin = torch.polar(torch.full_like(angle, factor), angle)
    y = x.clone()
    if case["interleaved"]:
        z = torch.view_as_complex(x[..., :rot].reshape(*x.shape[:-1], n, 2).contiguous()) * spin
        y[..., :rot] = torch.view_as_real(z).reshape(*x.shape[:-1], rot)
    else:
        z = torch.complex(x[..., :n].contiguous(), x[..., n:rot].contiguous()) * spin
        y[..., :n], y[..., n:rot] = z.real, z.imag
    return y


def _exact_diff(state):
    """A loop over sequences and heads; the gradients by automatic differentiation."""
    case = state["case"]
    b, h, hk = case["batch"], case["heads"], case["kv_heads"]
    train = case["train"]
    names = ("q", "k", "v", "lam")
    x = {n: state[n].double() for n in names}
    grads = {n: torch.zeros_like(x[n]) for n in names}
    out = torch.zeros(b, case["tokens"], h, case["dv"], dtype=torch.float64, device=DEVICE)
    lengths = _lengths(case)
    i = torch.arange(case["tokens"], device=DEVICE)[:, None]
    for n in range(b):
        if not lengths[n]:
            continue
        j = torch.arange(lengths[n], device=DEVICE)[None, :]
        seen = (j <= i + case["start"]) if case["causal"] else torch.ones_like(i + j, dtype=torch.bool)
        for head in range(h):
            kv = head // (h // hk)
            part = [x["q"][n, :, 2 * head : 2 * head + 2], x["k"][n, : lengths[n], 2 * kv : 2 * kv + 2],
                    x["v"][n, : lengths[n], kv], x["lam"][head]]
            part = [p.detach().clone().requires_grad_(train) for p in part]
            logits = torch.einsum("tmd,smd->mts", part[0], part[1]) / math.sqrt(case["d"])
            weights = torch.exp(logits - torch.logsumexp(logits.masked_fill(~seen, float("-inf")), -1, keepdim=True)) * seen
            y = weights[0] @ part[2] - part[3] * (weights[1] @ part[2])
            out[n, :, head] = y.detach()
            if train:
                got = torch.autograd.grad(y, part, state["dout"][n, :, head].double())
                grads["q"][n, :, 2 * head : 2 * head + 2] += got[0]
                grads["k"][n, : lengths[n], 2 * kv : 2 * kv + 2] += got[1]
                grads["v"][n, : lengths[n], kv] += got[2]
                grads["lam"][head] += got[3]
            del logits, weights, y
    return [out] + [grads[n] for n in names] if train else [out]


def exact(case, seed):
    state = prepare(case, seed)
    if case["op"] == "diff":
        return _exact_diff(state)
    if case["op"] == "rotary":
        x = state["x"].double().requires_grad_(case["train"])
        leaves, outputs, seeds = [x], [_exact_turn(x, state)], ["dy"]
    else:
        leaves = [state[n].double().requires_grad_(case["train"]) for n in ("q", "k", "q_weight", "k_weight")]
        outputs = []
        for x, weight in ((leaves[0], leaves[2]), (leaves[1], leaves[3])):
            norm = torch.sqrt(x.square().sum(-1, keepdim=True) / case["dim"] + EPS)
            outputs.append(_exact_turn(x / norm * weight, state))
        seeds = ["dq", "dk"]
    if not case["train"]:
        return outputs
    grads = torch.autograd.grad(outputs, leaves, [state[n].double() for n in seeds])
    return [y.detach() for y in outputs] + list(grads)
