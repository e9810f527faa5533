"""The operators of a block around a selective state space, as cases that can be timed and compared.

``scan_train``     the selective scan over whole sequences, forward and backward: the temporal mixer of a training step.
``scan_forward``   the same without gradients, state in and out: (chunked) prefill and evaluation.
``scan_step``      one token per row, the state updated in place: generation.
``conv_train``     the short causal convolution with its activation in front of the scan, forward and backward.
``conv_step``      the same for one token per row, the window updated in place.
``norm_train``     the residual's addition and the norm in front of the block, forward and backward.
``norm_bytes``     the same without gradients, rows in 8 bits with a scale each, for a product in 8 bits.

``own`` chooses between the calls that a program makes of the package and plain PyTorch in 32 bits.

The selective scan carries N numbers for each channel w, which reads and writes the vectors B, C of its group:

    h_t[n] = exp(s_t A[n]) h_{t-1}[n] + s_t u_t B_t[n],  s_t = softplus(dt_t + dt_bias),  y_t = (sum_n C_t[n] h_t[n] + D u_t) silu(z_t)

A reset discards the history in front of its token; an inactive token leaves the state as it is and gives zeros.
"""

import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6


def _scan(kind, batch, steps, width, states, groups=1, dtype="bf16", tokens="all", carried=False, gated=True):
    return {"kind": kind, "batch": batch, "steps": steps, "width": width, "states": states, "groups": groups, "dtype": dtype,
            "tokens": tokens, "carried": carried, "gated": gated}


def _conv(kind, batch, steps, width, taps, dtype="bf16", tokens="all", carried=False, activation="silu"):
    return {"kind": kind, "batch": batch, "steps": steps, "width": width, "taps": taps, "dtype": dtype, "tokens": tokens,
            "carried": carried, "activation": activation}


def _norm(kind, rows, width, dtype="bf16", residual="bf16"):
    return {"kind": kind, "rows": rows, "width": width, "dtype": dtype, "residual": residual}


def listed():
    named = {
        # a training step at the package's training shape (8 rows of 2048 tokens, width 1024), the mixer twice as wide as the block
        "scan train B8 T2048 W2048 N16": _scan("scan_train", 8, 2048, 2048, 16),
        # packed documents with padding behind them, odd sizes, two groups, in full precision, behind a carried state
        "scan train packed B3 T777 W180 f32": _scan("scan_train", 3, 777, 180, 12, groups=2, dtype="f32", tokens="packed", carried=True),
        # one long prompt at a width of 2560: few rows, so the sequence itself has to fill the device
        "scan prefill B1 T16384 W2560": _scan("scan_forward", 1, 16384, 2560, 16),
        # the next short piece of a few prompts behind a cache
        "scan prefill B3 T137 W1024": _scan("scan_forward", 3, 137, 1024, 16, carried=True),
        # one token for each sequence of a large serving batch
        "scan step B256 W2048": _scan("scan_step", 256, 1, 2048, 16),
        # generation for a single user: the smallest call of all
        "scan step B1 W2048": _scan("scan_step", 1, 1, 2048, 16),
        # the convolution of the training step
        "conv train B8 T2048 W2048 K4": _conv("conv_train", 8, 2048, 2048, 4),
        # packed documents, odd sizes, full precision
        "conv train packed B3 T777 W180 f32": _conv("conv_train", 3, 777, 180, 3, dtype="f32", tokens="packed", carried=True),
        # the convolution of a decode step, some rows idle
        "conv step B256 W2048": _conv("conv_step", 256, 1, 2048, 4, tokens="packed"),
        # the norm in front of the block at the training shape, the residual stream in full precision
        "norm train 16384x1024": _norm("norm_train", 16384, 1024, residual="f32"),
        # a prompt's rows for a product in 8 bits
        "norm bytes 16384x2560": _norm("norm_bytes", 16384, 2560),
        # the rows of a decode step
        "norm bytes 64x1024": _norm("norm_bytes", 64, 1024),
    }
    return [dict(c, name=name) for name, c in named.items()]


def _spread(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["scan_train", "scan_train", "scan_forward", "scan_step", "conv_train", "conv_step", "norm_train", "norm_bytes"])
    dtype = rng.choice(["bf16", "bf16", "f32"])
    tokens, carried = rng.choice(["all", "packed"]), rng.random() < 0.5
    if kind.startswith("norm"):
        width = rng.choice([1024, 2560, 8 * rng.randint(4, 512), rng.randint(1, 1000)])
        return _norm(kind, _spread(rng, 1, (1 << 23) // width), width, dtype, rng.choice([dtype, "f32"]))
    width = rng.choice([1024, 2048, 8 * rng.randint(4, 256), rng.randint(16, 1000)])
    if kind.startswith("conv"):
        steps = 1 if kind == "conv_step" else _spread(rng, 1, 4096)
        batch = _spread(rng, 1, max(1, min(256, (1 << 22) // (steps * width))))
        return _conv(kind, batch, steps, width, rng.choice([4, 4, 3, 2]), dtype, tokens, carried, rng.choice(["silu", "silu", "none"]))
    states = rng.choice([16, 16, 8, 32, 64, rng.randint(1, 64)])
    groups = rng.choice([g for g in (1, 1, 2, 4) if width % g == 0])
    steps = 1 if kind == "scan_step" else _spread(rng, 1, 4096)
    batch = _spread(rng, 1, max(1, min(256, (1 << 27) // (steps * width * states))))
    return _scan(kind, batch, steps, width, states, groups, dtype, tokens, carried, rng.random() < 0.7)


def work(case):
    kind, es = case["kind"], 2 if case["dtype"] == "bf16" else 4
    if kind.startswith("norm"):
        n, rs = case["rows"] * case["width"], 2 if case["residual"] == "bf16" else 4
        if kind == "norm_bytes":
            return {"bytes": (es + 2 * rs + 1) * n + 4 * case["rows"], "flops": 7 * n}
        # forward: x and the residual in, both results out; backward: the sum and both upstream gradients in, one gradient for each addend out
        return {"bytes": (es + 2 * rs + es + rs + es + rs + es + rs) * n, "flops": 16 * n}
    tokens = case["batch"] * case["steps"]
    n = tokens * case["width"]
    if kind == "conv_step":
        return {"bytes": es * n * (2 + 2 * (case["taps"] - 1)), "flops": n * (2 * case["taps"] + 4)}
    if kind == "conv_train":
        return {"bytes": 5 * es * n, "flops": n * (6 * case["taps"] + 12)}    # x, y; x, dy, dx
    vectors, streams = 2 * tokens * case["groups"] * case["states"], 4 if case["gated"] else 3
    state = case["batch"] * case["width"] * case["states"]
    moved = es * (streams * n + vectors) + 4 * state                          # u, dt, z, y, B, C and the last state
    flops = (7 * case["states"] + 16) * n
    if case["carried"] or kind == "scan_step":
        moved += 4 * state
    if kind == "scan_train":
        moved += es * ((2 * streams - 1) * n + 2 * vectors) + (4 * state if case["carried"] else 0)   # u, dt, z, dy, B, C again, their gradients
        flops += (20 * case["states"] + 40) * n
    return {"bytes": moved, "flops": flops}


# ---- inputs ------------------------------------------------------------------------------------------------------
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
    dtype, train = DTYPES[case["dtype"]], case["kind"].endswith("_train")

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=gen)

    def leaf(t):
        return t.requires_grad_(train)

    if case["kind"].startswith("norm"):
        rows, width, residual = case["rows"], case["width"], DTYPES[case["residual"]]
        leaves = [leaf(normal(rows, width).to(dtype)), leaf((3 * normal(rows, width)).to(residual)), leaf((0.1 * normal(width)).to(dtype))]
        ups = [normal(rows, width).to(dtype), normal(rows, width).to(residual)] if train else None
        return {"case": case, "leaves": leaves, "ups": ups}
    batch, steps, width = case["batch"], case["steps"], case["width"]
    reset, active = _masks(case, gen)
    flags = None if reset is None else reset[:, 0].to(torch.uint8) + 2 * (~active[:, 0]).to(torch.uint8)
    made = {"case": case, "reset": reset, "active": active, "flags": flags}
    if case["kind"].startswith("conv"):
        taps = case["taps"]
        both = normal(batch, steps, 2 * width).to(dtype)                       # one projection: what is convolved, and the gate
        weight, bias = (normal(width, 1, taps) / math.sqrt(taps)).to(dtype), (0.2 * normal(width)).to(dtype)
        window = normal(batch, taps - 1, width).to(dtype)
        if case["kind"] == "conv_step":
            return dict(made, args=[both[:, 0, :width], weight, bias], window=window)
        leaves = [leaf(both[..., :width]), leaf(weight), leaf(bias)] + ([leaf(window)] if case["carried"] else [])
        return dict(made, leaves=leaves, up=normal(batch, steps, width).to(dtype) if train else None)
    states, groups = case["states"], case["groups"]
    u = torch.nn.functional.silu(normal(batch, steps, width)).to(dtype)        # behind the convolution
    dt = (0.7 * normal(batch, steps, width)).to(dtype)
    rate = 0.001 * 100 ** torch.rand(width, device="cuda", generator=gen)      # step sizes of 0.001 to 0.1
    dt_bias = rate + torch.log(-torch.expm1(-rate))
    A = -torch.arange(1, states + 1, device="cuda") * torch.exp(0.1 * normal(width, states))
    one = normal(batch, steps, 8 + 2 * groups * states).to(dtype)              # one projection: a low-rank part, B and C
    B, C = (one[..., 8 + k * groups * states:8 + (k + 1) * groups * states].unflatten(-1, (groups, states)) for k in (0, 1))
    z = normal(batch, steps, 2 * width).to(dtype)[..., width:] if case["gated"] else None
    D = 1 + 0.1 * normal(width)
    state = 0.3 * normal(batch, width, states) if case["carried"] or case["kind"] == "scan_step" else None
    if case["kind"] == "scan_step":
        return dict(made, args=[t[:, 0] for t in (u, dt)] + [A] + [t[:, 0] for t in (B, C)], state=state, D=D, dt_bias=dt_bias,
                    z=None if z is None else z[:, 0])
    names = {"u": u, "dt": dt, "A": A, "B": B, "C": C, "D": D, "z": z, "dt_bias": dt_bias, "h0": state}
    leaves = {name: leaf(t) for name, t in names.items() if t is not None}
    return dict(made, leaves=leaves, up=normal(batch, steps, width).to(dtype) if train else None)


# ---- the plain forms ---------------------------------------------------------------------------------------------
def _softplus(x):
    return torch.clamp(x, min=0) + torch.log1p(torch.exp(-x.abs()))


def _sigmoid(x):
    return 1 / (1 + torch.exp(-x))


def _linear_recurrence(decay, added):
    """h_t = decay_t h_{t-1} + added_t along axis 1, by doubling."""
    shift = 1
    while shift < added.shape[1]:
        added = torch.cat((added[:, :shift], added[:, shift:] + decay[:, shift:] * added[:, :-shift]), 1)
        decay = torch.cat((decay[:, :shift], decay[:, shift:] * decay[:, :-shift]), 1)
        shift *= 2
    return added


def _scan_plain(leaves, reset, active, up):
    """(out, last state), or with an upstream gradient (out, gradients in the order of the leaves)."""
    f = {name: t.detach().float() for name, t in leaves.items()}
    batch, steps, width = f["u"].shape
    groups, states = f["B"].shape[2:]

    def live(t):
        return t if active is None else torch.where(active.reshape(batch, steps, *[1] * (t.dim() - 2)), t, 0.0)

    def split(t):                                                              # [B, T, W] -> [B, T, G, W / G, 1]
        return t.reshape(batch, steps, groups, width // groups, 1)

    def joined(t):
        return t.reshape(batch, steps, width)

    def per_channel(t):                                                        # [W, N] -> [G, W / G, N]
        return t.reshape(groups, width // groups, -1)

    def per_group(t):                                                          # [B, T, G, N] -> [B, T, G, 1, N]
        return t[:, :, :, None]

    pre = live(f["dt"] + f["dt_bias"])
    u, s, B, C, A = split(live(f["u"])), split(live(_softplus(pre))), per_group(live(f["B"])), per_group(live(f["C"])), per_channel(f["A"])
    z = None if "z" not in f else split(live(f["z"]))
    starts = None if reset is None else (reset if active is None else reset & active).reshape(batch, steps, 1, 1, 1)
    decay = torch.exp(s * A)
    if starts is not None:
        decay = torch.where(starts, 0.0, decay)
    added = s * u * B
    if "h0" in f:
        h0 = f["h0"].reshape(batch, groups, width // groups, states)
        added[:, 0] += decay[:, 0] * h0
    h = _linear_recurrence(decay, added)
    y = (C * h).sum(-1, keepdim=True) + per_channel(f["D"][:, None]) * u
    gate = None if z is None else z * _sigmoid(z)
    out = live(joined(y if z is None else y * gate))
    if up is None:
        return out, h[:, -1].reshape(batch, width, states)
    del added
    dout = split(live(up.float()))
    dy = dout if z is None else dout * gate
    # what a state's gradient takes from the token behind it: the recurrence again, from the end
    later = torch.cat((decay[:, 1:], torch.zeros_like(decay[:, :1])), 1)
    dh = _linear_recurrence(later.flip(1), (C * dy).flip(1)).flip(1)
    del later
    first = torch.zeros_like(h[:, :1]) if "h0" not in f else h0[:, None]
    through = dh * decay * torch.cat((first, h[:, :-1]), 1)                    # gradient at the exponent
    along = (dh * B).sum(-1, keepdim=True)
    ds = (through * A).sum(-1, keepdim=True) + u * along
    ddt = live(joined(ds) * _sigmoid(pre))
    grads = {
        "u": live(joined(s * along + per_channel(f["D"][:, None]) * dy)), "dt": ddt,
        "A": (through * s).sum((0, 1)).reshape(width, states), "B": live((dh * (s * u)).sum(3)), "C": live((h * dy).sum(3)),
        "D": joined(dy * u).sum((0, 1)), "dt_bias": ddt.sum((0, 1)),
    }
    if z is not None:
        rising = _sigmoid(z)
        grads["z"] = live(joined(dout * y * rising * (1 + z * (1 - rising))))
    if "h0" in f:
        grads["h0"] = (dh[:, 0] * decay[:, 0]).reshape(batch, width, states)
    return out, [grads[name] for name in leaves]


def _scan_step_plain(args, D, z, dt_bias, state, flags):
    u, dt, A, B, C = (t.float() for t in args)
    s = _softplus(dt + dt_bias)[..., None]
    share = u.shape[1] // B.shape[1]
    B, C = (t.repeat_interleave(share, 1) for t in (B, C))
    new = torch.exp(s * A) * state
    idle = None
    if flags is not None:
        idle = (flags & 2) != 0
        new = torch.where((flags & 1).bool()[:, None, None], 0.0, new)
    new = new + s * u[..., None] * B
    out = (new * C).sum(-1) + D * u
    if z is not None:
        out = out * z.float() * _sigmoid(z.float())
    if idle is not None:
        new, out = torch.where(idle[:, None, None], state, new), torch.where(idle[:, None], 0.0, out)
    state.copy_(new)
    return out


def _sources(case, reset, active, window):
    """For every token and lag the place of its tap's input in cat(window, x) (the K - 1 rows of the window first), and whether there is
    one: taps go back over the active tokens of the document."""
    batch, steps, back = case["batch"], case["steps"], case["taps"] - 1
    device = "cuda"
    active = torch.ones(batch, steps, dtype=torch.bool, device=device) if active is None else active
    reset = torch.zeros_like(active) if reset is None else reset & active
    live = torch.cat((torch.ones(batch, back, dtype=torch.bool, device=device), active), 1)
    document = torch.cat((torch.zeros(batch, back, dtype=torch.long, device=device), reset.long().cumsum(1)), 1)
    rank = live.long().cumsum(1) - 1                                           # how many active tokens lie in front
    place = torch.zeros(batch, back + steps, dtype=torch.long, device=device)
    at = torch.arange(back + steps, device=device).expand(batch, -1)
    place.scatter_(1, torch.where(live, rank, back + steps - 1), torch.where(live, at, 0))
    lags = torch.arange(back + 1, device=device)
    wanted = rank[:, back:, None] - lags                                       # [B, T, K]
    source = place.gather(1, wanted.clamp(min=0).flatten(1)).reshape(wanted.shape)
    inside = (wanted >= 0) & active[..., None] & (document.gather(1, source.flatten(1)).reshape(source.shape) == document[:, back:, None])
    if not window:
        inside &= source >= back
    return source, inside, live, rank


def _conv_plain(state, up):
    """out, or with an upstream gradient (out, gradients in the order of the leaves)."""
    case, leaves = state["case"], state["leaves"]
    batch, steps, width, back = case["batch"], case["steps"], case["width"], case["taps"] - 1
    x, weight, bias = (t.detach().float() for t in leaves[:3])
    rows = x if len(leaves) < 4 and back == 0 else torch.cat((x.new_zeros(batch, back, width) if len(leaves) < 4 else leaves[3].detach().float(), x), 1)
    source, inside, _, _ = _sources(case, state["reset"], state["active"], len(leaves) > 3)
    at = torch.arange(batch, device="cuda")[:, None, None]
    taken = torch.where(inside[..., None], rows[at, source], 0.0)              # [B, T, K, W], by lag
    taps = weight[:, 0].flip(1).T                                              # by lag
    pre = (taken * taps).sum(2) + bias
    live = None if state["active"] is None else state["active"][..., None]
    rising = _sigmoid(pre)
    out = pre * rising if case["activation"] == "silu" else pre
    out = out if live is None else torch.where(live, out, 0.0)
    if up is None:
        return out
    dpre = up.float() * (rising * (1 + pre * (1 - rising)) if case["activation"] == "silu" else 1.0)
    dpre = dpre if live is None else torch.where(live, dpre, 0.0)
    drows = torch.zeros_like(rows)
    drows.scatter_add_(1, source.flatten(1)[..., None].expand(-1, -1, width), (torch.where(inside[..., None], dpre[:, :, None] * taps, 0.0)).flatten(1, 2))
    dweight = (taken * dpre[:, :, None]).sum((0, 1)).T.flip(1)[:, None]
    grads = [drows[:, back:], dweight, dpre.sum((0, 1))]
    return out, grads + ([drows[:, :back]] if len(leaves) > 3 else [])


def _conv_step_plain(args, window, flags, activation):
    x, weight, bias = (t.float() for t in args)
    old = window.float()
    if flags is not None:
        old = torch.where((flags == 1)[:, None, None], 0.0, old)
    rows = torch.cat((old, x[:, None]), 1)
    out = (rows * weight[:, 0].T).sum(1) + bias
    out = out * _sigmoid(out) if activation == "silu" else out
    new = rows[:, 1:]
    if flags is not None:
        idle = (flags & 2) != 0
        out, new = torch.where(idle[:, None], 0.0, out), torch.where(idle[:, None, None], window.float(), new)
    window.copy_(new)
    return out


def _norm_plain(leaves, ups):
    x, residual, g = (t.detach().float() for t in leaves)
    total = (x + residual).to(leaves[1].dtype)                                 # the stream as it is stored
    s = total.float()
    inverse = 1 / (s.square().mean(-1, keepdim=True) + EPS).sqrt()
    y = s * inverse * (1 + g)
    if ups is None:
        return y, total
    scaled = ups[0].float() * (1 + g)
    ds = inverse * (scaled - s * inverse.square() * (scaled * s).mean(-1, keepdim=True)) + ups[1].float()
    return y, total, [ds, ds, (ups[0].float() * s * inverse).sum(0)]


def _to_bytes(y):
    scale = y.abs().amax(-1, keepdim=True).clamp(min=2.0 ** -100) / 448
    return (y / scale).to(torch.float8_e4m3fn), scale


def _as_leaves(grads, leaves):
    return [g.to(t.dtype) for g, t in zip(grads, leaves)]


def run(state):
    case, kind = state["case"], state["case"]["kind"]
    train = kind.endswith("_train")
    if own:
        import griffin_amd
    if kind == "norm_train":
        leaves = state["leaves"]
        if own:
            outs = griffin_amd.hip_add_rmsnorm(*leaves, EPS)
            return [t.detach() for t in outs], torch.autograd.grad(outs, leaves, state["ups"])
        y, total, grads = _norm_plain(leaves, state["ups"])
        return [y.to(leaves[0].dtype), total], _as_leaves(grads, leaves)
    if kind == "norm_bytes":
        if own:
            return griffin_amd.hip_add_rmsnorm_quantised(*state["leaves"], EPS)
        y, total = _norm_plain(state["leaves"], None)
        return *_to_bytes(y), total
    if kind == "conv_step":
        activation = None if case["activation"] == "none" else case["activation"]
        if own:
            return griffin_amd.hip_short_conv_step(*state["args"], state["window"], activation, state["flags"]), state["window"]
        return _conv_step_plain(state["args"], state["window"], state["flags"], activation).to(state["args"][0].dtype), state["window"]
    if kind == "conv_train":
        leaves = state["leaves"]
        if own:
            activation, window = None if case["activation"] == "none" else case["activation"], leaves[3] if len(leaves) > 3 else None
            out, _ = griffin_amd.hip_short_conv(*leaves[:3], window, activation, state["reset"], state["active"], need_state=False)
            return out.detach(), torch.autograd.grad(out, leaves, state["up"])
        out, grads = _conv_plain(state, state["up"])
        return out.to(leaves[0].dtype), _as_leaves(grads, leaves)
    if kind == "scan_step":
        if own:
            return griffin_amd.hip_selective_step(*state["args"], state["state"], state["D"], state["z"], state["dt_bias"],
                                                  flags=state["flags"]), state["state"]
        out = _scan_step_plain(state["args"], state["D"], state["z"], state["dt_bias"], state["state"], state["flags"])
        return out.to(state["args"][0].dtype), state["state"]
    leaves = state["leaves"]
    if own:
        out, last = griffin_amd.hip_selective_scan(**leaves, reset_mask=state["reset"], active_mask=state["active"])
        return (out.detach(), torch.autograd.grad(out, list(leaves.values()), state["up"])) if train else (out, last)
    out, rest = _scan_plain(leaves, state["reset"], state["active"], state["up"])
    return out.to(leaves["u"].dtype), _as_leaves(rest, leaves.values()) if train else rest


# ---- from the definitions, in 64 bits ----------------------------------------------------------------------------
def _exact_scan(state, train):
    leaves = {name: t.detach().double() for name, t in state["leaves"].items()}
    u, dt, A, B, C = (leaves[n] for n in ("u", "dt", "A", "B", "C"))
    batch, steps, width = u.shape
    group = torch.arange(width, device="cuda") // (width // B.shape[2])
    x = dt + leaves["dt_bias"]
    s = torch.nn.functional.softplus(x, threshold=60)
    z, D = leaves.get("z"), leaves["D"]
    reset, active = state["reset"], state["active"]
    h = leaves.get("h0", torch.zeros(batch, width, A.shape[1], device="cuda", dtype=torch.float64))
    before, y = [], torch.empty_like(u)

    def decay_of(t):
        a = torch.exp(s[:, t, :, None] * A)
        return a if reset is None else a.masked_fill(reset[:, t, None, None], 0.0)

    for t in range(steps):
        if train:
            before.append(h)
        new = decay_of(t) * h + (s[:, t] * u[:, t])[..., None] * B[:, t, group]
        y[:, t] = torch.linalg.vecdot(new, C[:, t, group]) + D * u[:, t]
        h = new if active is None else torch.where(active[:, t, None, None], new, h)
    on = torch.ones(batch, steps, 1, dtype=torch.float64, device="cuda") if active is None else active[..., None].double()
    sig = None if z is None else torch.sigmoid(z)
    out = on * (y if z is None else y * z * sig)
    if not train:
        return out, h
    dout = on * state["up"].double()
    dy = dout if z is None else dout * z * sig
    dB, dC, along, ds = (torch.zeros_like(t) for t in (B, C, u, u))
    dA, carry, spread = torch.zeros_like(A), torch.zeros_like(h), torch.nn.functional.one_hot(group).double().T
    for t in range(steps - 1, -1, -1):
        a, write = decay_of(t), (s[:, t] * u[:, t])[..., None] * B[:, t, group]
        now = a * before[t] + write
        dC[:, t] = torch.matmul(spread, now * dy[:, t, :, None])
        dh = carry + dy[:, t, :, None] * C[:, t, group]
        dh = dh if active is None else dh * on[:, t, :, None]
        dB[:, t] = torch.matmul(spread, dh * (s[:, t] * u[:, t])[..., None])
        along[:, t] = torch.linalg.vecdot(dh, B[:, t, group])
        kept = dh * a * before[t]
        dA += (kept * s[:, t, :, None]).sum(0)
        ds[:, t] = torch.linalg.vecdot(kept, A.expand_as(kept))
        carry = a * dh if active is None else torch.where(active[:, t, None, None], a * dh, carry)
    ddt = (ds + u * along) * torch.sigmoid(x)
    grads = {"u": s * along + D * dy, "dt": ddt, "A": dA, "B": dB, "C": dC, "D": (dy * u).sum((0, 1)), "dt_bias": ddt.sum((0, 1)), "h0": carry}
    if z is not None:
        grads["z"] = dout * y * sig * (1 + z * (1 - sig))
    return out, [grads[name] for name in leaves]


def _exact_scan_step(state):
    u, dt, A, B, C = (t.double() for t in state["args"])
    group = torch.arange(u.shape[1], device="cuda") // (u.shape[1] // B.shape[1])
    s = torch.nn.functional.softplus(dt + state["dt_bias"].double(), threshold=60)
    old = state["state"].double()
    on, fresh = (torch.full_like(u[:, :1], v) for v in (1.0, 0.0))
    if state["flags"] is not None:
        on, fresh = ((state["flags"] & 2) == 0)[:, None].double(), (state["flags"] & 1)[:, None].double()
    new = torch.exp(s[..., None] * A) * old * (1 - fresh)[..., None] + (s * u)[..., None] * B[:, group]
    out = torch.linalg.vecdot(new, C[:, group]) + state["D"].double() * u
    if state["z"] is not None:
        out = out * torch.nn.functional.silu(state["z"].double())
    return on * out, torch.where(on[..., None] > 0, new, old)


def _exact_conv(state):
    """Token by token: the window holds the last K - 1 active inputs of the document, the gradients walk back through it."""
    case, leaves = state["case"], [t.detach().double() for t in state["leaves"]]
    x, weight, bias = leaves[:3]
    batch, steps, width = x.shape
    back = case["taps"] - 1
    taps = weight[:, 0].T                                                      # oldest first
    window = x.new_zeros(batch, back, width) if len(leaves) < 4 else leaves[3]
    silu = case["activation"] == "silu"
    windows, pres = [], []
    for t in range(steps):
        old = window if state["reset"] is None else window.masked_fill(state["reset"][:, t, None, None], 0.0)
        rows = torch.cat((old, x[:, t, None]), 1)
        windows.append(rows)
        pres.append((rows * taps).sum(1) + bias)
        window = rows[:, 1:] if state["active"] is None else torch.where(state["active"][:, t, None, None], rows[:, 1:], window)
    pre = torch.stack(pres, 1)
    sig = torch.sigmoid(pre)
    on = torch.ones(batch, steps, 1, dtype=torch.float64, device="cuda") if state["active"] is None else state["active"][..., None].double()
    out = on * (pre * sig if silu else pre)
    dpre = on * state["up"].double() * (sig * (1 + pre * (1 - sig)) if silu else 1.0)
    dx, dtaps, dwindow = torch.zeros_like(x), torch.zeros_like(taps), torch.zeros_like(window)
    for t in range(steps - 1, -1, -1):
        drows = torch.cat((torch.zeros_like(dwindow[:, :1]), dwindow), 1)[:, -case["taps"]:] if back else torch.zeros_like(x[:, :1])
        drows = drows + dpre[:, t, None] * taps
        dtaps += (windows[t] * dpre[:, t, None]).sum(0)
        kept = drows[:, :back] if state["reset"] is None else drows[:, :back].masked_fill(state["reset"][:, t, None, None], 0.0)
        dx[:, t] = drows[:, back] if state["active"] is None else drows[:, back] * on[:, t]
        dwindow = kept if state["active"] is None else torch.where(state["active"][:, t, None, None], kept, dwindow)
    return out, [dx, dtaps.T[:, None], dpre.sum((0, 1))] + ([dwindow] if len(leaves) > 3 else [])


def _exact_conv_step(state):
    x, weight, bias = (t.double() for t in state["args"])
    old = state["window"].double()
    fresh, on = torch.zeros_like(x[:, :1]), torch.ones_like(x[:, :1])
    if state["flags"] is not None:
        fresh, on = (state["flags"] == 1)[:, None].double(), ((state["flags"] & 2) == 0)[:, None].double()
    rows = torch.cat((old * (1 - fresh)[..., None], x[:, None]), 1)
    out = torch.einsum("bkw,wk->bw", rows, weight[:, 0]) + bias
    out = torch.nn.functional.silu(out) if state["case"]["activation"] == "silu" else out
    return on * out, torch.where(on[..., None] > 0, rows[:, 1:], old)


def _exact_norm(state):
    x, residual, g = (t.detach().double() for t in state["leaves"])
    total = x + residual
    s = total.float().to(state["leaves"][1].dtype).double()                    # the sum as the stream holds it
    length = (s.square().mean(-1, keepdim=True) + EPS).sqrt()
    y = s / length * (1 + g)
    if state["case"]["kind"] == "norm_bytes":
        return None, y.abs().amax(-1, keepdim=True) / 448, total
    up = state["ups"][0].double()
    along = (up * (1 + g) * s).mean(-1, keepdim=True)
    ds = up * (1 + g) / length - s * along / length ** 3 + state["ups"][1].double()
    return [y, total], [ds, ds, (up * s / length).sum(0)]


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["kind"].startswith("norm"):
            return _exact_norm(state)
        if case["kind"] == "conv_step":
            return _exact_conv_step(state)
        if case["kind"] == "conv_train":
            return _exact_conv(state)
        if case["kind"] == "scan_step":
            return _exact_scan_step(state)
        return _exact_scan(state, case["kind"] == "scan_train")
