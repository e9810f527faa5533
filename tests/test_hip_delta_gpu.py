"""The gated delta rule on the GPU against its definition, token by token in 64 bits."""

import os
import subprocess
import sys

import pytest
import torch

from griffin_amd import hip_gated_delta, hip_gated_delta_step
from tests.helpers import rel_err

pytestmark = pytest.mark.gpu

NAMES = ("q", "k", "v", "log_decay", "beta", "h0")
BF16, F32 = torch.bfloat16, torch.float32
# Largest deviation over largest value.  fp32: sums of up to 128 products, each off by 2^-24, through two products in a row for a
# result and four for a gradient.  bf16: a result is rounded once, 2^-8; what is computed before enters the products
# to 2^-17, through up to eight of them in a row, which also bounds the fp32 states of bf16 operands.
OUT = {F32: 2 ** -16, BF16: 2 ** -8 + 2 ** -14}
GRAD = {F32: 2 ** -15, BF16: 2 ** -8 + 2 ** -13}
STATE = {F32: 2 ** -16, BF16: 2 ** -14}
STATE_GRAD = {F32: 2 ** -15, BF16: 2 ** -13}


def recurrence(q, k, v, log_decay, beta, h0, scale, reset=None, active=None):
    """o and the final state, from the definition (any float type, autograd works)."""
    B, T, H, K = q.shape
    HV, V = v.shape[2:]
    of = torch.arange(HV) // (HV // H)
    q, k = q[:, :, of], k[:, :, of]
    state = q.new_zeros(B, HV, K, V) if h0 is None else h0
    rows = []
    for t in range(T):
        kept = state * log_decay[:, t].exp()[..., None, None]
        if reset is not None:
            kept = torch.where(reset[:, t, None, None, None], torch.zeros_like(kept), kept)
        error = v[:, t] - (kept * k[:, t, :, :, None]).sum(2)
        new = kept + k[:, t, :, :, None] * (beta[:, t, :, None] * error)[:, :, None]
        out = scale * (new * q[:, t, :, :, None]).sum(2)
        if active is not None:
            live = active[:, t, None, None]
            new = torch.where(live[..., None], new, state)
            out = torch.where(live, out, torch.zeros_like(out))
        state = new
        rows.append(out)
    return torch.stack(rows, 1), state


def make(B, T, H, HV, K, V, dtype=F32, carried=True, seed=0, slow=False):
    gen = torch.Generator().manual_seed(seed)
    normal = lambda *shape: torch.randn(*shape, generator=gen)
    unit = lambda t: t / t.norm(dim=-1, keepdim=True)
    made = {
        "q": unit(normal(B, T, H, K)), "k": unit(normal(B, T, H, K) + 0.3), "v": normal(B, T, HV, V),
        "log_decay": -torch.nn.functional.softplus(normal(B, T, HV) - (6 if slow else 2)), "beta": torch.sigmoid(normal(B, T, HV)),
    }
    made = {name: t.to(dtype) for name, t in made.items()}
    made["h0"] = 0.5 * normal(B, HV, K, V) if carried else None
    made["up"], made["up_state"] = normal(B, T, HV, V).to(dtype), 0.2 * normal(B, HV, K, V)
    return made


def masks(B, T, seed=1):
    gen = torch.Generator().manual_seed(seed)
    reset = torch.rand(B, T, generator=gen) < 4.0 / T
    lengths = torch.randint(1, T + 1, (B,), generator=gen)
    return reset, torch.arange(T)[None] < lengths[:, None]


def run(fn, case, reset, active, device, dtype=None, scale=None):
    leaves = [None if case[n] is None else case[n].to(device=device, dtype=dtype or case[n].dtype).requires_grad_(True) for n in NAMES]
    put = lambda t: None if t is None else t.to(device)
    scale = case["q"].shape[-1] ** -0.5 if scale is None else scale
    out, last = fn(*leaves, scale, put(reset), put(active))
    wrt = [t for t in leaves if t is not None]
    grads = torch.autograd.grad([out, last], wrt, [case["up"].to(out), case["up_state"].to(last)])
    return out.detach(), last.detach(), dict(zip([n for n, t in zip(NAMES, leaves) if t is not None], grads))


def check(case, reset=None, active=None, scale=None):
    dtype = case["q"].dtype
    want, want_last, want_grads = run(recurrence, case, reset, active, "cpu", torch.float64, scale)
    got, last, grads = run(hip_gated_delta, case, reset, active, "cuda", None, scale)
    torch.cuda.synchronize()
    # as fp32 numbers: exp(-20000) is 2^-28853 in 64 bits and 0 in any result, whose smallest number is 2^-149
    want, want_last, want_grads = want.float(), want_last.float(), {n: t.float() for n, t in want_grads.items()}
    assert got.dtype == dtype and last.dtype == F32
    errors = {"o": rel_err(got, want) / OUT[dtype], "state": rel_err(last, want_last) / STATE[dtype]}
    for name in grads:
        assert grads[name].dtype == case[name].dtype and grads[name].shape == case[name].shape
        errors["d" + name] = rel_err(grads[name], want_grads[name]) / (STATE_GRAD if name == "h0" else GRAD)[dtype]
    assert all(e <= 1 for e in errors.values()), errors


SHAPES = [
    # B, T, H, HV, K, V: one token; one chunk; a token more; several chunks; odd sizes; shared key heads
    (1, 1, 1, 1, 8, 8),
    (2, 64, 2, 2, 32, 32),
    (2, 65, 1, 3, 40, 24),
    (1, 200, 2, 4, 128, 128),
    (3, 130, 2, 2, 96, 80),
    (1, 63, 1, 1, 128, 20),
    (2, 150, 1, 2, 100, 33),
    (1, 300, 1, 1, 64, 144),
    (1, 129, 1, 1, 1, 1),
    (1, 90, 3, 3, 17, 65),
]


@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_whole_sequences(shape, dtype):
    check(make(*shape, dtype=dtype, carried=shape[1] % 2 == 0))


@pytest.mark.parametrize("shape", [(3, 130, 2, 2, 96, 80), (4, 77, 1, 2, 64, 32), (2, 200, 2, 2, 128, 64)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_packed_documents_and_padding(shape, dtype):
    reset, active = masks(*shape[:2])
    case = make(*shape, dtype=dtype)
    check(case, reset, active)
    check(case, reset, None)
    check(case, None, active)


def test_every_token_a_document():
    check(make(2, 70, 1, 1, 32, 32), torch.ones(2, 70, dtype=torch.bool), None)


def test_masks_with_holes_and_rows_without_tokens():
    gen = torch.Generator().manual_seed(5)
    active = torch.rand(4, 140, generator=gen) < 0.5
    active[1] = False
    active[2, :64] = False
    reset = torch.rand(4, 140, generator=gen) < 0.1
    for dtype in (F32, BF16):
        check(make(4, 140, 1, 2, 64, 48, dtype=dtype), reset, active)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_masked_tokens_may_hold_anything(dtype):
    reset, active = masks(3, 130, seed=4)
    case = make(3, 130, 2, 4, 64, 64, dtype=dtype)
    clean = run(hip_gated_delta, case, reset, active, "cuda")
    for name in ("q", "k", "v", "log_decay", "beta", "up"):
        case[name] = case[name].clone()
        case[name][~active] = float("nan") if name != "log_decay" else float("inf")
    dirty = run(hip_gated_delta, case, reset, active, "cuda")
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])
    for name in NAMES:
        assert torch.equal(clean[2][name], dirty[2][name]), name
        if name != "h0":
            assert not dirty[2][name][~active.cuda()].any()
    assert not dirty[0][~active.cuda()].any()


def test_a_decay_of_nothing_is_a_reset():
    case = make(2, 100, 1, 2, 32, 32)
    reset = torch.zeros(2, 100, dtype=torch.bool)
    reset[:, 10] = reset[0, 64] = reset[1, 99] = True
    want = run(hip_gated_delta, case, reset, None, "cuda")
    case["log_decay"] = case["log_decay"].masked_fill(reset[..., None], -float("inf"))
    got = run(hip_gated_delta, case, None, None, "cuda")
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    for name in NAMES:
        assert torch.equal(got[2][name], want[2][name]), name


def test_decays_that_are_thousands_apart_in_a_chunk():
    """The running sum reaches thousands, where 32 bits no longer hold the differences between neighbours."""
    case = make(1, 128, 1, 1, 32, 32)
    case["log_decay"][:, ::2] = -300.0
    check(case)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_slow_decay_over_many_chunks(dtype):
    check(make(1, 700, 1, 1, 64, 64, dtype=dtype, slow=True))


@pytest.mark.parametrize("shape", [(1, 1500, 1, 2, 64, 48), (2, 1100, 1, 1, 128, 20), (1, 1290, 1, 1, 20, 100)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_long_sequences_of_few_heads(shape, dtype):
    """Walked in segments side by side, which are joined; slow decay carries the state across them."""
    check(make(*shape, dtype=dtype, slow=True))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_long_packed_sequences_of_few_heads(dtype):
    reset, active = masks(2, 1300, seed=3)
    active[0, 600:700] = False
    check(make(2, 1300, 1, 2, 64, 32, dtype=dtype, slow=True), reset, active)


def test_gates_in_another_type_than_the_activations():
    case = make(2, 100, 1, 2, 64, 64, dtype=BF16)
    case["log_decay"], case["beta"] = case["log_decay"].float(), case["beta"].float()
    check(case)
    case["beta"] = case["beta"].to(BF16)
    check(case)


def test_scale_is_a_factor_of_the_output():
    check(make(1, 80, 1, 1, 32, 32), scale=0.75)


@pytest.mark.parametrize("offset", [0, 3])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_parts_of_one_projection_are_read_in_place(dtype, offset):
    B, T, H, HV, K, V = 2, 100, 2, 4, 32, 24
    case = make(B, T, H, HV, K, V, dtype=dtype, carried=False)
    flat = torch.cat([case[n].reshape(B, T, -1) for n in "qkv"], -1)
    wide = torch.zeros(B, T, flat.shape[-1] + 2 * offset + 8, dtype=dtype)
    wide[..., offset:offset + flat.shape[-1]] = flat
    wide = wide.cuda().requires_grad_(True)
    q, k, v = wide[..., offset:offset + flat.shape[-1]].split([H * K, H * K, HV * V], -1)
    q, k, v = q.view(B, T, H, K), k.view(B, T, H, K), v.view(B, T, HV, V)
    gates = [case[n].cuda() for n in ("log_decay", "beta")]
    out, _ = hip_gated_delta(q, k, v, *gates)
    want, _ = hip_gated_delta(*(case[n].cuda() for n in NAMES[:5]))
    assert torch.equal(out, want)
    (grad,) = torch.autograd.grad(out, wide, case["up"].cuda())
    dense = run(hip_gated_delta, dict(case, up_state=torch.zeros(B, HV, K, V)), None, None, "cuda")[2]
    assert torch.equal(grad[..., offset:offset + flat.shape[-1]], torch.cat([dense[n].reshape(B, T, -1) for n in "qkv"], -1))


def test_pieces_with_a_carried_state_are_the_whole():
    case = {n: None if t is None else t.cuda() for n, t in make(2, 230, 1, 2, 64, 64).items()}
    reset, active = (m.cuda() for m in masks(2, 230, seed=9))
    operands = [case[n] for n in NAMES[:5]]
    whole, last = hip_gated_delta(*operands, case["h0"], reset_mask=reset, active_mask=active)
    state, rows = case["h0"], []
    for a, b in ((0, 1), (1, 64), (64, 65), (65, 200), (200, 230)):
        out, state = hip_gated_delta(*(t[:, a:b] for t in operands), state, reset_mask=reset[:, a:b], active_mask=active[:, a:b])
        rows.append(out)
    assert rel_err(torch.cat(rows, 1), whole) <= 2 * OUT[F32] and rel_err(state, last) <= 2 * STATE[F32]


@pytest.mark.parametrize("shape", [(3, 2, 4, 64, 64), (2, 1, 1, 128, 128), (5, 2, 2, 40, 33), (1, 1, 3, 7, 1), (2, 4, 4, 128, 200)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_single_tokens(shape, dtype):
    B, H, HV, K, V = shape
    T = 12
    case = make(B, T, H, HV, K, V, dtype=dtype)
    gen = torch.Generator().manual_seed(7)
    reset, active = torch.rand(B, T, generator=gen) < 0.2, torch.rand(B, T, generator=gen) < 0.8
    want, want_last = recurrence(*(case[n].double() for n in NAMES), K ** -0.5, reset, active)
    state = case["h0"].cuda()
    flags = (reset.to(torch.uint8) + 2 * (~active).to(torch.uint8)).cuda()
    outs = []
    for t in range(T):
        before = state.clone()
        outs.append(hip_gated_delta_step(*(case[n][:, t].cuda() for n in NAMES[:5]), state, flags=flags[:, t]))
        idle = ~active[:, t].cuda()
        assert torch.equal(state[idle], before[idle])
    assert rel_err(torch.stack(outs, 1), want) <= OUT[dtype]
    assert rel_err(state, want_last) <= 2 ** -16                # fp32 throughout, whatever the operands' type


def test_steps_behind_a_prompt():
    """A prompt in one call, then token by token, as generation runs it."""
    case = {n: None if t is None else t.cuda() for n, t in make(2, 80, 2, 4, 128, 64, dtype=BF16, carried=False).items()}
    operands = [case[n] for n in NAMES[:5]]
    whole, last = hip_gated_delta(*operands)
    _, state = hip_gated_delta(*(t[:, :70] for t in operands))
    outs = [hip_gated_delta_step(*(t[:, i] for t in operands), state) for i in range(70, 80)]
    assert rel_err(torch.stack(outs, 1), whole[:, 70:]) <= 2 * OUT[BF16] and rel_err(state, last) <= 2 * STATE[BF16]


def test_gradients_are_differences():
    """Central differences of the fp32 operator itself along random directions: h = 2^-6 leaves h^2 = 2^-12 of the third
    derivative and 2^-16 / h = 2^-10 of the results' own deviation."""
    case = make(1, 70, 1, 2, 16, 16)
    leaves = [case[n].cuda().requires_grad_(True) for n in NAMES]
    up, up_state = case["up"].cuda(), case["up_state"].cuda()

    def value(args):
        out, last = hip_gated_delta(*args)
        return ((out.double() * up.double()).sum() + (last.double() * up_state.double()).sum())

    grads = torch.autograd.grad(value(leaves), leaves)
    gen = torch.Generator().manual_seed(2)
    for i, (leaf, grad) in enumerate(zip(leaves, grads)):
        way = torch.randn(leaf.shape, generator=gen).cuda()
        way = way / way.norm()
        h = 2.0 ** -6
        with torch.no_grad():
            moved = [value([t if j != i else t + s * h * way for j, t in enumerate(leaves)]) for s in (1, -1)]
        difference = float((moved[0] - moved[1]) / (2 * h))
        along = float((grad.double() * way.double()).sum())
        assert abs(difference - along) <= 2 ** -8 * float(grad.double().norm()), NAMES[i]


def test_only_the_state_or_only_the_output_is_used():
    case = make(2, 100, 1, 1, 32, 32)
    leaves = [case[n].cuda().requires_grad_(True) for n in NAMES]
    full = run(hip_gated_delta, case, None, None, "cuda")[2]
    out, last = hip_gated_delta(*leaves)
    first = torch.autograd.grad(out, leaves, case["up"].cuda(), retain_graph=True)
    second = torch.autograd.grad(last, leaves, case["up_state"].cuda())
    for name, a, b in zip(NAMES, first, second):
        assert rel_err(a + b, full[name]) <= 2 * GRAD[F32], name
    with pytest.raises(RuntimeError):
        torch.autograd.grad(hip_gated_delta(*leaves)[0].sum(), leaves, create_graph=True)[0].sum().backward()


def test_other_stream_than_the_tensors():
    case = make(2, 100, 2, 2, 64, 64, dtype=BF16)
    want = run(hip_gated_delta, case, None, None, "cuda")
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = run(hip_gated_delta, case, None, None, "cuda")
    side.synchronize()
    assert torch.equal(got[0], want[0]) and all(torch.equal(got[2][n], want[2][n]) for n in NAMES)


def test_results_repeat_bit_for_bit():
    case = make(2, 300, 2, 4, 128, 64, dtype=BF16)
    first, second = (run(hip_gated_delta, case, None, None, "cuda") for _ in range(2))
    assert torch.equal(first[0], second[0]) and torch.equal(first[1], second[1])
    assert all(torch.equal(first[2][n], second[2][n]) for n in NAMES)


def test_a_state_that_is_carried_by_itself():
    """Sequences of one token, of masked tokens alone, and of nothing but the carried state."""
    case = make(2, 1, 1, 2, 32, 32)
    check(case)
    check(case, None, torch.zeros(2, 1, dtype=torch.bool))
    case = make(1, 130, 1, 1, 32, 32)
    check(case, None, torch.zeros(1, 130, dtype=torch.bool))


def test_a_reset_mask_that_is_written_between_calls():
    case = make(1, 100, 1, 1, 32, 32, carried=False)
    operands = [case[n].cuda() for n in NAMES[:5]]
    reset = torch.zeros(1, 100, dtype=torch.bool, device="cuda")
    plain, none = hip_gated_delta(*operands, reset_mask=reset), hip_gated_delta(*operands)
    assert torch.equal(plain[0], none[0])
    reset[0, 50] = True
    got, last = hip_gated_delta(*operands, reset_mask=reset)
    want, want_last = recurrence(*(t.cpu().double() for t in operands), None, 32 ** -0.5, reset.cpu())
    assert rel_err(got, want) <= OUT[F32] and rel_err(last, want_last) <= STATE[F32]
    with torch.inference_mode():
        made = reset.clone()
    leaves = [t.requires_grad_(True) for t in operands]
    torch.autograd.grad(hip_gated_delta(*leaves, reset_mask=made)[0].sum(), leaves)


def test_two_calls_at_once():
    """On two streams, in segments and not: nothing is shared."""
    cases = [make(1, 1500, 1, 1, 128, 64, dtype=BF16, seed=7), make(2, 300, 2, 4, 64, 64, dtype=BF16, seed=8)]
    want = [run(hip_gated_delta, case, None, None, "cuda") for case in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for stream, case in zip(streams, cases):
            with torch.cuda.stream(stream):
                got.append(run(hip_gated_delta, case, None, None, "cuda"))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1]) and all(torch.equal(a[2][n], b[2][n]) for n in NAMES)


def test_captures():
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    child = subprocess.run([sys.executable, "-u", "-m", "tests.capture_operators_child"], cwd=root, capture_output=True, text=True, timeout=100)
    print(child.stdout + child.stderr[-2000:], flush=True)
    assert child.returncode == 0


def test_states_that_go_past_the_caches():
    """Large batches, whose states are not kept in the caches, against the same rows in parts."""
    B, H, K, V = 260, 8, 128, 128                              # 130 MiB of state
    gen = torch.Generator("cuda").manual_seed(3)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    q, k = (torch.nn.functional.normalize(normal(B, H, K), dim=-1).bfloat16() for _ in range(2))
    rest = [normal(B, H, V).bfloat16(), -normal(B, H).abs(), normal(B, H).sigmoid()]
    flags = (torch.arange(B, device="cuda") % 5 == 0).to(torch.uint8)
    state = normal(B, H, K, V)
    parts = [[t[i : i + 65].clone() for t in (q, k, *rest, state, flags)] for i in range(0, B, 65)]
    out = hip_gated_delta_step(q, k, *rest, state, flags=flags)
    want = torch.cat([hip_gated_delta_step(*part[:6], flags=part[6]) for part in parts])
    assert torch.equal(out, want) and torch.equal(state, torch.cat([part[5] for part in parts]))

    case = make(8, 1100, 12, 12, 128, 128, dtype=BF16)        # 162 MiB of states and values
    whole = run(hip_gated_delta, case, None, None, "cuda")
    halves = [run(hip_gated_delta, {n: t[i : i + 4] for n, t in case.items()}, None, None, "cuda") for i in (0, 4)]
    assert rel_err(whole[0], torch.cat([h[0] for h in halves])) <= 2 * OUT[BF16]
    assert rel_err(whole[1], torch.cat([h[1] for h in halves])) <= 2 * STATE[BF16]
    for name in NAMES:
        assert rel_err(whole[2][name], torch.cat([h[2][name] for h in halves])) <= 2 * GRAD[BF16], name


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_broadcast_operands_and_gradients(dtype):
    """Operands that one number stands for along an axis, gradients that autograd hands over without memory of their own."""
    case = make(2, 90, 2, 2, 32, 48, dtype=dtype)
    case["q"] = case["q"][:, :1, :1]                           # one query for all tokens and heads
    case["beta"] = case["beta"][:1, :1, :1]

    def results(fn, device, to):
        leaves = [case[n].to(device=device, dtype=to or case[n].dtype).requires_grad_(True) for n in NAMES]
        q, k, v, log_decay, beta, h0 = leaves
        out, last = fn(q.expand(2, 90, 2, 32), k, v, log_decay, beta.expand(2, 90, 2), h0)
        return [out.detach(), last.detach(), *torch.autograd.grad(out.float().sum() + last.sum() if to is None else out.sum() + last.sum(), leaves)]

    want = results(lambda *t: recurrence(*t, 32 ** -0.5), "cpu", torch.float64)
    got = results(hip_gated_delta, "cuda", None)
    # a broadcast input's gradient is the sum of up to 360 of those of its uses, which cancel by less than sixteen to one
    for name, g, w in zip(("o", "state", *NAMES), got, want):
        limit = OUT[dtype] if name == "o" else STATE[dtype] if name == "state" else (16 if name in ("q", "beta") else 1) * GRAD[dtype]
        assert rel_err(g, w) <= limit, (name, rel_err(g, w))


def test_offsets_that_pass_32_bits():
    """A prompt of more than 2^31 elements a tensor and a state of as many: the ends by themselves give the same."""
    gen = torch.Generator("cuda").manual_seed(5)
    normal = lambda *shape, by=1.0: torch.empty(*shape, dtype=BF16, device="cuda").normal_(generator=gen).mul_(by)
    T, H, K, tail = (1 << 19) + 128, 32, 128, 128
    q, k, v = normal(1, T, H, K, by=K ** -0.5), normal(1, T, H, K, by=0.8 * K ** -0.5), normal(1, T, H, K)
    decay, beta = -normal(1, T, H).abs_(), normal(1, T, H).sigmoid_()
    out, last = hip_gated_delta(q, k, v, decay, beta)
    front = [t[:, : T - tail] for t in (q, k, v, decay, beta)]
    _, state = hip_gated_delta(*front)
    want, want_last = hip_gated_delta(*(t[:, T - tail :] for t in (q, k, v, decay, beta)), state)
    assert rel_err(out[:, T - tail :], want) <= 2 * OUT[BF16] and rel_err(last, want_last) <= 2 * STATE[BF16]
    del q, k, v, out, front

    B, H = 16500, 8
    state = torch.empty(B, H, K, K, device="cuda").normal_(generator=gen)
    token = [normal(B, H, K, by=K ** -0.5), normal(B, H, K, by=K ** -0.5), normal(B, H, K), -normal(B, H).abs_(), normal(B, H).sigmoid_()]
    end = state[-4:].clone()
    out = hip_gated_delta_step(*token, state)
    assert torch.equal(out[-4:], hip_gated_delta_step(*(t[-4:] for t in token), end)) and torch.equal(state[-4:], end)


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape, skipped", [((2, 1, 1, 2, 40, 33), 0), ((1, 1, 2, 2, 128, 128), 0), ((1, 71, 1, 1, 64, 64), 70), ((2, 200, 1, 1, 64, 64), 150)], ids=str)
def test_a_first_token_has_nothing_to_decay(shape, skipped, dtype):
    """The gradient of its log decay is zero, not a rounding: without a state in front, and behind padding."""
    case = make(*shape, dtype=dtype, carried=False)
    active = (torch.arange(shape[1]) >= skipped).expand(shape[0], -1) if skipped else None
    _, _, grads = run(hip_gated_delta, case, None, active, "cuda")
    assert grads["log_decay"][:, : skipped + 1].abs().max() == 0
    check(case, None, active)
    if shape[1] == 1:
        carried = make(*shape, dtype=dtype)
        assert run(hip_gated_delta, carried, None, None, "cuda")[2]["log_decay"].abs().min() > 0


@pytest.mark.parametrize("V", [40, 48, 80])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_masked_tokens_may_hold_anything_beside_any_width(V, dtype):
    """Behind the last columns of a value lie the next head's and, behind the last head, the next token's."""
    reset, active = masks(3, 130, seed=4)
    active[0] = torch.arange(130) < 37                          # padding behind the middle of a chunk
    case = make(3, 130, 2, 4, 64, V, dtype=dtype)
    clean = run(hip_gated_delta, case, reset, active, "cuda")
    for name in ("q", "k", "v", "log_decay", "beta", "up"):
        case[name] = case[name].clone()
        case[name][~active] = float("nan") if name != "log_decay" else float("inf")
    dirty = run(hip_gated_delta, case, reset, active, "cuda")
    assert torch.equal(clean[0], dirty[0]) and torch.equal(clean[1], dirty[1])
    for name in NAMES:
        assert torch.equal(clean[2][name], dirty[2][name]), name


@pytest.mark.parametrize("heads", [(2, 2), (2, 4)], ids=str)
@pytest.mark.parametrize("V", [33, 40, 48, 80])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_heads_keep_their_gradients_whatever_others_receive(V, dtype, heads):
    case = make(2, 70, *heads, 64, V, dtype=dtype)
    share = heads[1] // heads[0]
    clean = run(hip_gated_delta, case, None, None, "cuda")[2]
    for value in (float("inf"), float("nan")):
        for spoilt in range(2):                                 # the value heads of one key head
            of = slice(spoilt * share, (spoilt + 1) * share)
            case["up"] = case["up"].clone()
            kept = case["up"].clone()
            case["up"][:, :, of] = value
            got = run(hip_gated_delta, case, None, None, "cuda")[2]
            case["up"] = kept
            rest = slice((1 - spoilt) * share, (2 - spoilt) * share)
            for name in NAMES:
                axis = 1 if name == "h0" else 2
                one = slice(1 - spoilt, 2 - spoilt) if name in ("q", "k") else rest
                picked = [t[(slice(None),) * axis + (one,)] for t in (got[name], clean[name])]
                assert torch.equal(*picked), name


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_axes_of_one_element_may_have_any_stride(dtype):
    """A token of one row out of a projection whose rows are no whole vectors; tokens of a long way apart, of which there is one."""
    H, HV, K, V = 2, 4, 32, 24
    width = 2 * H * K + HV * V
    gen = torch.Generator().manual_seed(3)
    rows = torch.randn(1, 9, width + 2, generator=gen).to(dtype).cuda()
    gates = [-torch.rand(1, 1, HV, generator=gen).cuda(), torch.rand(1, 1, HV, generator=gen).cuda()]

    def both(views):
        results = []
        for operands in (views, [t.clone(memory_format=torch.contiguous_format) for t in views]):
            leaves = [t.detach().requires_grad_(True) for t in operands]
            batch = leaves[0].shape[0]
            out, last = hip_gated_delta(*leaves, *(g.expand(batch, 1, HV) for g in gates))
            results.append([out, last, *torch.autograd.grad(out.sum() + last.sum(), leaves)])
            with torch.no_grad():
                results[-1].append(hip_gated_delta(*leaves, *(g.expand(batch, 1, HV) for g in gates))[0])
        assert all(torch.equal(a, b) for a, b in zip(*results))

    for token in range(9):
        q, k, v = rows[:, token : token + 1, :width].split([H * K, H * K, HV * V], -1)
        both([q.view(1, 1, H, K), k.view(1, 1, H, K), v.view(1, 1, HV, V)])
    far = torch.randn(2 * 2 * H * K + 2 * HV * V, generator=gen).to(dtype).cuda()
    parts = far.split([2 * H * K, 2 * H * K, 2 * HV * V])
    both([t.as_strided((2, 1, heads, size), (heads * size, 1 << 23, size, 1), t.storage_offset())
          for t, heads, size in zip(parts, (H, H, HV), (K, K, V))])


@pytest.mark.parametrize("skipped", [0, 5, 64, 70])
@pytest.mark.parametrize("shape", [(2, 130, 1, 2, 64, 48), (1, 300, 2, 2, 128, 64), (1, 1500, 1, 1, 64, 40)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_a_first_document_discards_whatever_state_there_is(shape, skipped, dtype):
    """A recycled state in front of a document start, padding between them or not, walked in one or in segments."""
    case = make(*shape, dtype=dtype)
    B, T = shape[:2]
    active = (torch.arange(T) >= skipped).expand(B, T) if skipped else None
    reset = torch.zeros(B, T, dtype=torch.bool)
    reset[:, skipped] = True
    case["h0"] = torch.zeros_like(case["h0"])
    want = run(hip_gated_delta, case, reset, active, "cuda")
    for value in (float("nan"), float("inf")):
        case["h0"] = torch.full_like(case["h0"], value)
        got = run(hip_gated_delta, case, reset, active, "cuda")
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        for name in NAMES:
            assert torch.equal(got[2][name], want[2][name]), name
        with torch.no_grad():
            put = lambda t: None if t is None else t.cuda()
            out, last = hip_gated_delta(*(case[n].cuda() for n in NAMES), reset_mask=put(reset), active_mask=put(active))
            assert rel_err(out, want[0]) <= 2 * OUT[dtype] and rel_err(last, want[1]) <= 2 * STATE[dtype]


@pytest.mark.parametrize("shape, start", [((2, 190, 1, 2, 64, 48), 64), ((1, 1500, 1, 1, 64, 40), 704), ((1, 1500, 1, 1, 128, 64), 128)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_chunks_in_front_of_a_document_receive_nothing_from_it(shape, start, dtype):
    """A document that starts a chunk: its gradients, whatever they are, end there."""
    case = make(*shape, dtype=dtype)
    reset = torch.zeros(*shape[:2], dtype=torch.bool)
    reset[:, start] = True
    want = run(hip_gated_delta, case, reset, None, "cuda")[2]
    for value in (float("nan"), float("inf")):
        case["up"] = case["up"].clone()
        case["up"][:, start:] = value
        case["up_state"] = torch.full_like(case["up_state"], value)
        got = run(hip_gated_delta, case, reset, None, "cuda")[2]
        assert torch.equal(got["h0"], want["h0"])
        for name in NAMES[:5]:
            assert torch.equal(got[name][:, :start], want[name][:, :start]), name


@pytest.mark.parametrize("shape", [(2, 130, 1, 2, 64, 48), (1, 1500, 1, 1, 64, 40)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_rows_without_tokens_keep_whatever_state_they_have(shape, dtype):
    case = make(*shape, dtype=dtype)
    active = torch.zeros(*shape[:2], dtype=torch.bool)
    for value in (None, float("nan"), float("inf")):
        if value is not None:
            case["h0"] = torch.full_like(case["h0"], value)
        out, last, grads = run(hip_gated_delta, case, None, active, "cuda")
        assert not out.any() and all(not grads[name].any() for name in NAMES[:5])
        assert rel_err(grads["h0"], case["up_state"]) <= STATE_GRAD[dtype]
        assert rel_err(last, case["h0"]) <= STATE[dtype] if value is None else not last.isfinite().any()
    case["up_state"] = torch.full_like(case["up_state"], float("nan"))
    grads = run(hip_gated_delta, case, None, active, "cuda")[2]
    assert all(not grads[name].any() for name in NAMES[:5]) and grads["h0"].isnan().all()


@pytest.mark.parametrize("heads", [(2, 2), (1, 3)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_documents_of_a_chunk_do_not_share_decay_gradients(dtype, heads):
    """A document without an upstream gradient has none of its decays, to the last bit."""
    T, starts = 128, (20, 41, 100)
    case = make(2, T, *heads, 64, 48, dtype=dtype)
    reset = torch.zeros(2, T, dtype=torch.bool)
    reset[:, list(starts)] = True
    whole, state = case["up"], case["up_state"]
    edges = (0, *starts, T)
    for a, b in zip(edges, edges[1:]):
        case["up"] = whole.clone()
        case["up"][:, a:b] = 0
        case["up_state"] = state if b < T else torch.zeros_like(state)
        grad = run(hip_gated_delta, case, reset, None, "cuda")[2]["log_decay"]
        assert not grad[:, a:b].any(), (a, b)
        assert grad.any()
        check(case, reset)


@pytest.mark.parametrize("heads", [(2, 2), (1, 2)], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_decay_gradients_where_little_is_left(dtype, heads):
    """Decays of e^-12 a token: what crosses a token is the write of the one in front of it, 2^-17 of what the tokens exchange with
    themselves.  A token's gradient is the product of the state that it keeps with that state's gradient and known to what those are
    known to (STATE, STATE_GRAD) of their norms' product, and to its own rounding."""
    case = make(2, 100, *heads, 64, 48, dtype=dtype)
    case["log_decay"] = (case["log_decay"].float() - 12.0).to(dtype)
    leaves = {n: case[n].double().requires_grad_(n == "log_decay") for n in NAMES}
    B, T, H, K = case["q"].shape
    of = torch.arange(heads[1]) // (heads[1] // heads[0])
    q, k = leaves["q"][:, :, of], leaves["k"][:, :, of]
    state, outs, kept = leaves["h0"], [], []
    for t in range(T):
        kept.append(state * leaves["log_decay"][:, t].exp()[..., None, None])
        kept[-1].retain_grad()
        error = leaves["v"][:, t] - (kept[-1] * k[:, t, :, :, None]).sum(2)
        state = kept[-1] + k[:, t, :, :, None] * (leaves["beta"][:, t, :, None] * error)[:, :, None]
        outs.append(K ** -0.5 * (state * q[:, t, :, :, None]).sum(2))
    ((torch.stack(outs, 1) * case["up"].double()).sum() + (state * case["up_state"].double()).sum()).backward()
    norm = lambda t: t.square().sum((-1, -2)).sqrt()
    product = torch.stack([norm(s.detach()) * norm(s.grad) for s in kept], 1)
    want = leaves["log_decay"].grad
    got = run(hip_gated_delta, case, None, None, "cuda")[2]["log_decay"].cpu().double()
    limit = (STATE[dtype] + STATE_GRAD[dtype]) * product + (2 ** -8 if dtype == BF16 else 2 ** -24) * want.abs()
    assert ((got - want).abs() / limit).max() <= 1, float(((got - want).abs() / limit).max())


def test_more_rows_than_a_launch_holds():
    """Single tokens of 2^23 rows, two workgroups each, against the step written out; keys of more than 2^32 elements in rows of whole vectors."""
    B, K, V = (1 << 23) + 5, 2, 33
    gen = torch.Generator("cuda").manual_seed(6)
    normal = lambda *shape: torch.empty(*shape, dtype=BF16, device="cuda").normal_(generator=gen)
    q, k, v, decay, beta = normal(B, 1, K), normal(B, 1, K), normal(B, 1, V), -normal(B, 1).abs_(), normal(B, 1).sigmoid_()
    state = torch.empty(B, 1, K, V, device="cuda").normal_(generator=gen)
    flags = (torch.arange(B, device="cuda") % 3).to(torch.uint8)
    for at in (slice(0, 1000), slice(B - 1000, B)):
        kept = state[at].double()
        out = hip_gated_delta_step(*(t[at] for t in (q, k, v, decay, beta)), state[at].clone(), flags=flags[at])
        qd, kd, vd = (t[at].double() for t in (q, k, v))
        kept = kept * torch.where(flags[at] == 1, 0.0, decay[at, 0].double().exp())[:, None, None, None]
        change = beta[at].double()[..., None] * (vd - (kept * kd[..., None]).sum(2))
        want = K ** -0.5 * ((kept + kd[..., None] * change[:, :, None]) * qd[..., None]).sum(2)
        assert rel_err(out, torch.where(flags[at] == 2, 0.0, want.movedim(0, -1)).movedim(-1, 0)) <= OUT[BF16]
    ends = [(at, state[at].clone()) for at in (slice(0, 1000), slice((1 << 23) - 500, B))]
    out = hip_gated_delta_step(q, k, v, decay, beta, state, flags=flags)
    for at, end in ends:
        assert torch.equal(out[at], hip_gated_delta_step(*(t[at] for t in (q, k, v, decay, beta)), end, flags=flags[at]))
        assert torch.equal(state[at], end)
    del state, out, q, k, v

    T, H, K, V = (1 << 20) + 64, 40, 100, 8
    q = normal(1, T, H, K).mul_(0.1)
    k, v, decay, beta = q.flip(-1), normal(1, T, H, V), normal(1, T, H).abs_().add_(1).neg_(), normal(1, T, H).sigmoid_()
    with torch.no_grad():
        out, last = hip_gated_delta(q, k, v, decay, beta)
    # decays of at least e^-1 a token: what is 128 tokens back is gone; three heads by the definition
    tail = [t[:, -192:, :3].double() for t in (q, k, v, decay, beta)]
    want, want_last = recurrence(*(t.cpu() for t in tail), None, K ** -0.5)
    assert rel_err(out[:, -64:, :3], want[:, -64:]) <= OUT[BF16] and rel_err(last[:, :3], want_last) <= STATE[BF16]


def test_large_passes_against_the_definition():
    """Sizes whose states go past the caches, of walks of two waves and of four: a row and its gradients by the definition."""
    for shape, row in (((8, 1408, 8, 8, 128, 128), 3), ((10, 1100, 8, 8, 128, 128), 9)):
        case = make(*shape, dtype=BF16)
        out, last, grads = run(hip_gated_delta, case, None, None, "cuda")
        one = {n: t[row : row + 1] for n, t in case.items()}
        want, want_last, want_grads = run(recurrence, one, None, None, "cuda", torch.float64)
        assert rel_err(out[row : row + 1], want) <= OUT[BF16] and rel_err(last[row : row + 1], want_last) <= STATE[BF16]
        for name in NAMES:
            assert rel_err(grads[name][row : row + 1], want_grads[name]) <= (STATE_GRAD if name == "h0" else GRAD)[BF16], name


def test_large_steps_against_the_definition():
    B, H, HV, K, V = 512, 4, 8, 128, 128                       # 256 MiB of state
    gen = torch.Generator("cuda").manual_seed(8)
    normal = lambda *shape: torch.randn(*shape, generator=gen, device="cuda")
    q, k = (torch.nn.functional.normalize(normal(B, H, K), dim=-1).bfloat16() for _ in range(2))
    v, decay, beta = normal(B, HV, V).bfloat16(), -normal(B, HV).abs(), normal(B, HV).sigmoid()
    state = normal(B, HV, K, V)
    of = torch.arange(HV, device="cuda") // (HV // H)
    kept = state.double() * decay.double().exp()[..., None, None]
    keys, queries = k.double()[:, of], q.double()[:, of]
    new = kept + keys[..., None] * (beta.double()[..., None] * (v.double() - (kept * keys[..., None]).sum(2)))[:, :, None]
    out = hip_gated_delta_step(q, k, v, decay, beta, state)
    assert rel_err(out, K ** -0.5 * (new * queries[..., None]).sum(2)) <= OUT[BF16] and rel_err(state, new) <= 2 ** -16


def test_the_end_of_a_long_prompt_against_the_definition():
    """More than 2^31 elements a tensor; decays of at least e^-1 a token leave nothing of what is 128 tokens back."""
    T, H, K, heads = (1 << 19) + 128, 32, 128, 4
    gen = torch.Generator("cuda").manual_seed(9)
    normal = lambda *shape, by=1.0: torch.empty(*shape, dtype=BF16, device="cuda").normal_(generator=gen).mul_(by)
    operands = [normal(1, T, H, K, by=K ** -0.5), normal(1, T, H, K, by=0.8 * K ** -0.5), normal(1, T, H, K),
                -normal(1, T, H).abs_().add_(1), normal(1, T, H).sigmoid_()]
    out, last = hip_gated_delta(*operands)
    tail = [t[:, -192:, -heads:].double().cpu() for t in operands]
    want, want_last = recurrence(*tail, None, K ** -0.5)
    assert rel_err(out[:, -64:, -heads:], want[:, -64:]) <= OUT[BF16] and rel_err(last[:, -heads:], want_last) <= STATE[BF16]


@pytest.mark.parametrize("T", [63, 200])
def test_what_parallel_keys_all_but_erase(T):
    """Keys of one element are parallel: a chunk erases nearly all of a state's gradient, whose terms are the upstream gradients of all tokens.
    Of those it is known to what a gradient of bf16 operands is (STATE_GRAD), not of the little that is left."""
    case = make(1, T, 1, 2, 1, 48, dtype=BF16, slow=True)
    _, _, want = run(recurrence, case, None, None, "cpu", torch.float64)
    _, _, grads = run(hip_gated_delta, case, None, None, "cuda")
    # a token hands on its query times its upstream gradient, both keys of one; what they erase of it comes back in the products
    q, up = case["q"].double(), case["up"].double()
    terms = (q[..., 0].abs().repeat(1, 1, 2)[..., None] * up.abs()).sum(1) + case["up_state"].double().abs()[:, :, 0]
    assert float(want["h0"].abs().max()) < 2 ** -4 * float(terms.max())
    assert ((grads["h0"].cpu().double() - want["h0"])[:, :, 0].abs() <= STATE_GRAD[BF16] * terms).all()
