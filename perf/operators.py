"""The operators around a matrix-valued recurrence, as cases that can be timed and compared.

``delta_train``    gated delta rule over whole sequences, forward and backward: the temporal mixer of a training step.
``delta_forward``  the same without gradients, state in and out: (chunked) prefill and evaluation.
``delta_step``     one token per row, the state updated in place: generation.
``norm_train``     group norm with an activation over channels-last features, forward and backward.
``norm_forward``   the same without gradients.

``own`` chooses between the calls that a program makes of the package and plain PyTorch in 32 bits.

The gated delta rule carries a [dk, dv] state S for each value head (a value head reads the key head of its group):

    S_t = a_t (I - beta_t k_t k_t') S_{t-1} + beta_t k_t v_t',    o_t = scale S_t' q_t,    a_t = exp(log_decay_t)

A reset discards the history in front of its token (a = 0); an inactive token leaves the state as it is and gives zeros.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
CHUNK = 64


def _delta(kind, batch, steps, heads, value_heads, dk, dv, dtype="bf16", tokens="all", carried=False):
    return {"kind": kind, "batch": batch, "steps": steps, "heads": heads, "value_heads": value_heads, "dk": dk, "dv": dv,
            "dtype": dtype, "tokens": tokens, "carried": carried}


def _norm(kind, batch, positions, channels, groups, activation, dtype="bf16"):
    return {"kind": kind, "batch": batch, "positions": positions, "channels": channels, "groups": groups,
            "activation": activation, "dtype": dtype}


def listed():
    named = {
        # a training step at the package's training shape: 8 rows of 2048 tokens, a width of 1024 as 8 heads of 128
        "delta train B8 T2048 H8": _delta("delta_train", 8, 2048, 8, 8, 128, 128),
        # a small layer in full precision: toy-model sized training
        "delta train small f32": _delta("delta_train", 2, 256, 4, 4, 64, 64, dtype="f32"),
        # packed documents with padding behind them, ragged length, two value heads to a key head, a carried state
        "delta train packed B3 T777": _delta("delta_train", 3, 777, 4, 8, 96, 80, tokens="packed", carried=True),
        # one long prompt, a width of 2560 as 20 heads: few rows, so the sequence itself has to fill the device
        "delta prefill B1 T32768 H20": _delta("delta_forward", 1, 32768, 20, 20, 128, 128),
        # the next short piece of a few prompts behind a cache
        "delta prefill B3 T137 H8": _delta("delta_forward", 3, 137, 8, 8, 128, 128, carried=True),
        # one token for each sequence of a large serving batch
        "delta step B256 H8": _delta("delta_step", 256, 1, 8, 8, 128, 128),
        # generation for a single user: the smallest call there is
        "delta step B1 H8": _delta("delta_step", 1, 1, 8, 8, 128, 128),
        # full precision, odd head sizes, three value heads to a key head, some rows idle
        "delta step odd B37 f32": _delta("delta_step", 37, 1, 4, 12, 72, 40, dtype="f32", tokens="packed"),
        # the heads' norm behind the mixer at the training shape: every token on its own, one group a head
        "norm train heads 16384x1024": _norm("norm_train", 16384, 1, 1024, 8, "none"),
        # features of a sequence normalised over its positions, at the same size
        "norm train B8 L2048 C1024": _norm("norm_train", 8, 2048, 1024, 32, "silu"),
        # odd sizes in full precision
        "norm train odd f32": _norm("norm_train", 3, 777, 180, 6, "gelu", dtype="f32"),
        # the heads' norm of a decode step
        "norm heads of a step": _norm("norm_forward", 256, 1, 1024, 8, "silu"),
    }
    return [dict(c, name=name) for name, c in named.items()]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["delta_train", "delta_train", "delta_forward", "delta_step", "norm_train", "norm_forward"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    if kind.startswith("delta"):
        heads = rng.choice([1, 2, 4, 6, 8])
        value_heads = heads * rng.choice([1, 1, 2, 3])
        dk, dv = (rng.choice([128, 64, 8 * rng.randint(3, 16), rng.randint(20, 128)]) for _ in range(2))
        tokens, carried = rng.choice(["all", "packed"]), rng.random() < 0.5
        if kind == "delta_step":
            return _delta(kind, _spread(rng, 1, 128 if value_heads <= 8 else 40), 1, heads, value_heads, dk, dv, dtype, tokens)
        steps = _spread(rng, 1, 4096)
        most = 16384 * 8 // (steps * value_heads) // (1 if dtype == "bf16" else 4)
        batch = _spread(rng, 1, max(1, min(8, most)))
        return _delta(kind, batch, steps, heads, value_heads, dk, dv, dtype, tokens, carried)
    groups = rng.choice([1, 4, 6, 8, 16, 32])
    channels = groups * rng.choice([16, 32, 64, 128, rng.randint(3, 100)])
    while channels > 2048:
        channels //= 2
    groups = next(g for g in (groups, 8, 4, 2, 1) if channels % g == 0)
    positions = rng.choice([1, _spread(rng, 2, 4096)])
    batch = _spread(rng, 1, max(1, (1 << 23) // (positions * channels)))
    return _norm(kind, batch, positions, channels, groups, rng.choice(["none", "silu", "gelu"]), dtype)


def work(case):
    es = 2 if case["dtype"] == "bf16" else 4
    if case["kind"].startswith("norm"):
        n = case["batch"] * case["positions"] * case["channels"]
        streams = 4 if case["kind"] == "norm_train" else 2                    # x, y; dy, dx
        return {"bytes": streams * es * n, "flops": (30 if case["kind"] == "norm_train" else 10) * n}
    tokens = case["batch"] * case["steps"]
    keys, values = 2 * case["heads"] * case["dk"], case["value_heads"] * case["dv"]
    gates = 2 * case["value_heads"]
    state = case["batch"] * case["value_heads"] * case["dk"] * case["dv"]
    moved = es * tokens * (keys + 2 * values + gates)                          # q, k, v, o, both gates
    flops = 6 * tokens * case["value_heads"] * case["dk"] * case["dv"]
    if case["kind"] == "delta_train":
        moved += es * tokens * (keys + 2 * values + gates)                     # dq, dk, do, dv and the gates' gradients
        moved += 8 * state if case["carried"] else 0
        flops += 14 * tokens * case["value_heads"] * case["dk"] * case["dv"]
    else:
        moved += 4 * state * (2 if case["carried"] or case["kind"] == "delta_step" else 1)
    return {"bytes": moved, "flops": flops}


# ---- inputs ------------------------------------------------------------------------------------------------------
def _unit(x):
    return x / (x.square().sum(-1, keepdim=True) + 1e-6).sqrt()


def _masks(case, gen):
    """Documents packed into rows: starts anywhere, padding behind the last one (rows of one token: some rows idle)."""
    batch, steps = case["batch"], case["steps"]
    if case["tokens"] == "all":
        return None, None
    starts = torch.rand(batch, steps, device="cuda", generator=gen) < 4.0 / max(steps, 8)
    lengths = steps - (torch.rand(batch, device="cuda", generator=gen) * 0.4 * steps).round().long()
    if steps == 1:
        lengths = (torch.rand(batch, device="cuda", generator=gen) < 0.8).long()
    return starts, torch.arange(steps, device="cuda")[None] < lengths[:, None]


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    train = case["kind"].endswith("_train")
    if case["kind"].startswith("norm"):
        shape = (case["batch"], case["positions"], case["channels"])
        x = (normal(*shape) + 0.5 * normal(shape[0], 1, shape[2])).to(dtype)
        weight, bias = (1 + 0.1 * normal(shape[2])).to(dtype), (0.1 * normal(shape[2])).to(dtype)
        leaves = [t.requires_grad_(train) for t in (x, weight, bias)]
        return {"case": case, "leaves": leaves, "up": normal(*shape).to(dtype) if train else None}
    batch, steps, h, hv, dk, dv = (case[n] for n in ("batch", "steps", "heads", "value_heads", "dk", "dv"))
    silu = torch.nn.functional.silu                                            # behind a short convolution, normalised
    q, k = (_unit(silu(normal(batch, steps, h, dk))).to(dtype) for _ in range(2))
    v = silu(normal(batch, steps, hv, dv)).to(dtype)
    rate = 16 ** torch.rand(hv, device="cuda", generator=gen)                  # decay rates of the heads, 1 to 16
    log_decay = (-rate * torch.nn.functional.softplus(normal(batch, steps, hv) - 4.0)).to(dtype)
    beta = torch.sigmoid(normal(batch, steps, hv)).to(dtype)
    state = 0.3 * normal(batch, hv, dk, dv) if case["carried"] or case["kind"] == "delta_step" else None
    reset, active = _masks(case, gen)
    made = {"case": case, "scale": dk ** -0.5, "reset": reset, "active": active, "state": state}
    if case["kind"] == "delta_step":
        flags = None if reset is None else reset[:, 0].to(torch.uint8) + 2 * (~active[:, 0]).to(torch.uint8)
        return dict(made, args=[t[:, 0].contiguous() for t in (q, k, v, log_decay, beta)], flags=flags)
    leaves = [q, k, v, log_decay, beta] + ([] if state is None else [state])
    leaves = [t.requires_grad_(train) for t in leaves]
    return dict(made, leaves=leaves, up=normal(batch, steps, hv, dv).to(dtype) if train else None)


# ---- the plain forms ---------------------------------------------------------------------------------------------
def _inverse(strict):
    """(I + strict)^-1 of strictly lower triangular [..., 64, 64] matrices: diagonal blocks of 1, 2, 4, ... joined in pairs."""
    size = strict.shape[-1]
    blocks = torch.ones(*strict.shape[:-2], size, 1, 1, dtype=strict.dtype, device=strict.device)
    half = 1
    while half < size:
        pairs = size // (2 * half)
        below = strict.reshape(*strict.shape[:-2], pairs, 2 * half, pairs, 2 * half).diagonal(dim1=-4, dim2=-2)
        below = below.movedim(-1, -3)[..., half:, :half]
        first, second = blocks[..., 0::2, :, :], blocks[..., 1::2, :, :]
        joined = -torch.matmul(torch.matmul(second, below), first)
        blocks = torch.cat((torch.cat((first, torch.zeros_like(first)), -1), torch.cat((joined, second), -1)), -2)
        half *= 2
    return blocks[..., 0, :, :]


def _delta_plain(q, k, v, log_decay, beta, state, scale, reset, active):
    batch, steps, hv = beta.shape
    if active is None:
        active = torch.ones(batch, steps, dtype=torch.bool, device=q.device)
    reset = torch.zeros_like(active) if reset is None else reset & active
    count = -(-steps // CHUNK)
    share = hv // q.shape[2]

    def chunks(t, live):                                                       # [B, T, H, ...] -> [B, H, chunk, token, ...]
        t = torch.where(live.reshape(batch, steps, *[1] * (t.dim() - 2)), t, torch.zeros((), dtype=t.dtype, device=t.device))
        t = torch.cat((t, t.new_zeros(batch, count * CHUNK - steps, *t.shape[2:])), 1)
        return t.reshape(batch, count, CHUNK, *t.shape[2:]).movedim(3, 1)

    q, k = (chunks(t.float(), active).repeat_interleave(share, 1) for t in (q, k))
    v, beta = chunks(v.float(), active), chunks(beta.float(), active)
    total = chunks(log_decay.double(), active & ~reset).cumsum(-1)             # far positions differ by little: 64 bits
    segment = chunks(reset[..., None].long(), active).cumsum(-1)
    lower = torch.ones(CHUNK, CHUNK, dtype=torch.bool, device=q.device).tril()
    joined = (segment[..., :, None] == segment[..., None, :]) & lower
    decay = (total[..., :, None] - total[..., None, :]).masked_fill(~joined, -math.inf).exp().float()
    write = decay * beta[..., None, :]
    solve = _inverse((torch.matmul(k, k.mT) * write).tril(-1))
    within = scale * torch.matmul(q, k.mT) * write
    from_start = total.masked_fill(segment != 0, -math.inf).exp().float()[..., None]
    to_end = (total[..., -1:] - total).masked_fill(segment != segment[..., -1:], -math.inf).exp().float()[..., None]
    keys_read, queries = from_start * k, scale * from_start * q
    keys_written = (to_end * beta[..., None] * k).mT
    state = torch.zeros(batch, hv, q.shape[-1], v.shape[-1], device=q.device) if state is None else state
    rows = []
    for n in range(count):
        z = torch.matmul(solve[:, :, n], v[:, :, n] - torch.matmul(keys_read[:, :, n], state))
        rows.append(torch.matmul(queries[:, :, n], state) + torch.matmul(within[:, :, n], z))
        state = from_start[:, :, n, -1:] * state + torch.matmul(keys_written[:, :, n], z)
    out = torch.stack(rows, 2).reshape(batch, hv, count * CHUNK, -1)[:, :, :steps].movedim(1, 2)
    return out, state


def _step_plain(q, k, v, log_decay, beta, state, scale, flags):
    share = beta.shape[1] // q.shape[1]
    q, k = (t.float().repeat_interleave(share, 1) for t in (q, k))
    v, decay, strength = v.float(), log_decay.float().exp(), beta.float()
    if flags is not None:
        idle, fresh = (flags & 2) != 0, flags == 1
        decay = torch.where(fresh[:, None], 0.0, torch.where(idle[:, None], 1.0, decay))
        strength = torch.where(idle[:, None], 0.0, strength)
        q = torch.where(idle[:, None, None], 0.0, q)
    kept = decay[..., None, None] * state
    change = strength[..., None] * (v - (kept * k[..., None]).sum(-2))
    state.copy_(kept + k[..., None] * change[..., None, :])
    return scale * (state * q[..., None]).sum(-2), state


def _gelu(t):
    return 0.5 * t * (1 + torch.tanh(math.sqrt(2 / math.pi) * (t + 0.044715 * t * t * t)))


def _norm_plain(x, weight, bias, groups, activation, eps):
    batch, positions, channels = x.shape
    x = x.float().reshape(batch, positions, groups, channels // groups)
    centred = x - x.mean((1, 3), keepdim=True)
    normed = centred / (centred.square().mean((1, 3), keepdim=True) + eps).sqrt()
    out = normed.reshape(batch, positions, channels) * weight.float() + bias.float()
    return out / (1 + torch.exp(-out)) if activation == "silu" else _gelu(out) if activation == "gelu" else out


EPS = 1e-5


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    train = kind.endswith("_train")
    if own:
        import griffin_amd
    if kind.startswith("norm"):
        x, weight, bias = state["leaves"]
        activation = case["activation"]
        if own:
            out = griffin_amd.hip_group_norm(x, case["groups"], weight, bias, EPS, None if activation == "none" else activation)
        else:
            out = _norm_plain(x, weight, bias, case["groups"], activation, EPS).to(x.dtype)
        if not train:
            return out
        return out.detach(), torch.autograd.grad(out, state["leaves"], state["up"])
    if kind == "delta_step":
        if own:
            out = griffin_amd.hip_gated_delta_step(*state["args"], state["state"], scale=state["scale"], flags=state["flags"])
            return out, state["state"]
        out, new = _step_plain(*state["args"], state["state"], state["scale"], state["flags"])
        return out.to(state["args"][2].dtype), new
    leaves = state["leaves"]
    operands, carried = leaves[:5], leaves[5] if len(leaves) > 5 else None
    if own:
        out, last = griffin_amd.hip_gated_delta(*operands, carried, scale=state["scale"], reset_mask=state["reset"],
                                                active_mask=state["active"])
    else:
        out, last = _delta_plain(*operands, carried, state["scale"], state["reset"], state["active"])
        out = out.to(operands[2].dtype)
    if not train:
        return out, last
    return out.detach(), torch.autograd.grad(out, leaves, state["up"])


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------
def _exact_delta(state, train):
    leaves = [t.detach().double() for t in state["leaves"]]
    q, k, v, log_decay, beta = leaves[:5]
    batch, steps, hv = beta.shape
    heads, dk, dv = q.shape[2], q.shape[3], v.shape[3]
    of = torch.arange(hv, device="cuda") // (hv // heads)
    q, k = state["scale"] * q[:, :, of], k[:, :, of]
    s = torch.zeros(batch, hv, dk, dv, device="cuda", dtype=torch.float64) if len(leaves) < 6 else leaves[5]
    decay = log_decay.exp()
    live = torch.ones(batch, steps, 1, device="cuda", dtype=torch.float64)
    if state["reset"] is not None:
        decay = decay.masked_fill(state["reset"][..., None], 0.0)
    if state["active"] is not None:
        live = state["active"][..., None].double()
        decay = decay.masked_fill(~state["active"][..., None], 1.0)
    beta, q = beta * live, q * live[..., None]
    out = torch.empty(batch, steps, hv, dv, device="cuda", dtype=torch.float64)
    before = torch.empty(steps, batch, hv, dk, dv, device="cuda", dtype=torch.float64) if train else None
    errors = torch.empty_like(out) if train else None
    for t in range(steps):
        if train:
            before[t] = s
        s = s * decay[:, t, :, None, None]
        error = v[:, t] - torch.matmul(k[:, t, :, None], s)[:, :, 0]
        s = s + k[:, t, :, :, None] * (beta[:, t, :, None] * error)[:, :, None]
        out[:, t] = torch.matmul(q[:, t, :, None], s)[:, :, 0]
        if train:
            errors[:, t] = error
    if not train:
        return out, s
    up = state["up"].double() * live[..., None]
    dq, dk_, dv_, dg, db = (torch.empty_like(t) for t in (q, k, v, beta, beta))
    ds = torch.zeros_like(s)
    for t in range(steps - 1, -1, -1):
        kept = before[t] * decay[:, t, :, None, None]
        error, strength = errors[:, t], beta[:, t, :, None]
        now = kept + k[:, t, :, :, None] * (strength * error)[:, :, None]
        dq[:, t] = torch.matmul(now, up[:, t, :, :, None])[..., 0]
        ds = ds + q[:, t, :, :, None] * up[:, t, :, None]
        along = torch.matmul(k[:, t, :, None], ds)[:, :, 0]                   # gradient of what the token wrote
        db[:, t] = (along * error).sum(-1)
        derror = strength * along
        dv_[:, t] = derror
        dk_[:, t] = torch.matmul(ds, (strength * error)[..., None])[..., 0] - torch.matmul(kept, derror[..., None])[..., 0]
        ds = ds - k[:, t, :, :, None] * derror[:, :, None]
        dg[:, t] = (ds * kept).sum((-1, -2))
        ds = ds * decay[:, t, :, None, None]
    if state["reset"] is not None:
        dg = dg.masked_fill(state["reset"][..., None], 0.0)

    def heads_of(d):
        return d.reshape(batch, steps, heads, hv // heads, dk).sum(3)

    grads = [heads_of(dq * live[..., None]) * state["scale"], heads_of(dk_ * live[..., None]), dv_ * live[..., None], dg * live, db * live]
    return out, tuple(grads + ([ds] if len(leaves) > 5 else []))


def _exact_step(state):
    q, k, v, log_decay, beta = (t.double().cpu().numpy() for t in state["args"])
    s = state["state"].double().cpu().numpy()
    out = v * 0
    flags = None if state["flags"] is None else state["flags"].cpu().numpy()
    for b in range(v.shape[0]):
        flag = 0 if flags is None else int(flags[b])
        if flag & 2:
            continue
        for h in range(v.shape[1]):
            key, query = (t[b, h * t.shape[1] // v.shape[1]] for t in (k, q))
            kept = s[b, h] * (0.0 if flag & 1 else math.exp(log_decay[b, h]))
            s[b, h] = kept + beta[b, h] * key[:, None] * (v[b, h] - key @ kept)[None]
            out[b, h] = state["scale"] * (query @ s[b, h])
    return out, s


def _exact_norm(state, train):
    case = state["case"]
    x, weight, bias = (t.detach().double() for t in state["leaves"])
    batch, positions, channels = x.shape
    groups, activation = case["groups"], case["activation"]
    split = x.reshape(batch, positions, groups, -1)
    variance, mean = torch.var_mean(split, (1, 3), correction=0, keepdim=True)
    inverse = (variance + EPS).rsqrt()
    normed = ((split - mean) * inverse).reshape(x.shape)
    pre = normed * weight + bias
    if activation == "silu":
        gate = torch.sigmoid(pre)
        out, slope = pre * gate, gate * (1 + pre * (1 - gate))
    elif activation == "gelu":
        inner = math.sqrt(2 / math.pi) * (pre + 0.044715 * pre ** 3)
        out = 0.5 * pre * (1 + inner.tanh())
        slope = 0.5 * (1 + inner.tanh()) + 0.5 * pre / inner.cosh() ** 2 * math.sqrt(2 / math.pi) * (1 + 3 * 0.044715 * pre ** 2)
    else:
        out, slope = pre, torch.ones_like(pre)
    if not train:
        return out
    dpre = state["up"].double() * slope
    dnormed = (dpre * weight).reshape(split.shape)
    like = normed.reshape(split.shape)
    dx = inverse * (dnormed - dnormed.mean((1, 3), keepdim=True) - like * (dnormed * like).mean((1, 3), keepdim=True))
    return out, (dx.reshape(x.shape), (dpre * normed).sum((0, 1)), dpre.sum((0, 1)))


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"].startswith("norm"):
        return _exact_norm(state, case["kind"] == "norm_train")
    if case["kind"] == "delta_step":
        return _exact_step(state)
    with torch.no_grad():
        return _exact_delta(state, case["kind"] == "delta_train")
