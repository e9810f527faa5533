"""Group norm with an activation on the GPU against its definition in 64 bits, and behind the gated delta rule."""

import pytest
import torch
import torch.nn.functional as F

from griffin_amd import hip_gated_delta, hip_gelu_gate, hip_group_norm
from tests.helpers import rel_err

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
# Largest deviation over largest value.  fp32: a sum is added up in runs of under 128 terms, each off by 2^-24, and its terms cancel by
# less than eight to one; the activations add 2^-20.  bf16: a result is rounded once, 2^-8.
TOLERANCE = {F32: 2 ** -16, BF16: 2 ** -8 + 2 ** -14}


def definition(x, groups, weight, bias, eps, activation):
    """Any float type, autograd works."""
    n, channels = x.shape[0], x.shape[-1]
    split = x.reshape(n, -1, groups, channels // groups)
    mean = split.mean((1, 3), keepdim=True)
    normed = (split - mean) / ((split - mean).square().mean((1, 3), keepdim=True) + eps).sqrt()
    out = normed.reshape(x.shape)
    if weight is not None:
        out = out * weight
    if bias is not None:
        out = out + bias
    return F.silu(out) if activation == "silu" else F.gelu(out, approximate="tanh") if activation == "gelu" else out


def make(shape, dtype=F32, seed=0, params=(True, True), far=0.0):
    gen = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=gen)
    x = (normal(*shape) + 0.5 * normal(shape[-1]) + far).to(dtype)
    weight = (1 + 0.2 * normal(shape[-1])).to(dtype) if params[0] else None
    bias = (0.3 * normal(shape[-1])).to(dtype) if params[1] else None
    return x, weight, bias, normal(*shape).to(dtype)


def run(fn, case, groups, eps, activation, device, dtype=None):
    *leaves, up = (None if t is None else t.to(device=device, dtype=dtype or t.dtype) for t in case)
    leaves = [None if t is None else t.requires_grad_(True) for t in leaves]
    out = fn(leaves[0], groups, leaves[1], leaves[2], eps, activation)
    return [out.detach(), *torch.autograd.grad(out, [t for t in leaves if t is not None], up)]


def check(case, groups, activation=None, eps=1e-5, tolerance=None):
    want = run(definition, case, groups, eps, activation, "cpu", torch.float64)
    got = run(hip_group_norm, case, groups, eps, activation, "cuda")
    errors = [rel_err(g, w) for g, w in zip(got, want)]
    assert all(g.dtype == case[0].dtype for g in got)
    assert max(errors) <= (tolerance or TOLERANCE[case[0].dtype]), errors


@pytest.mark.parametrize("shape, groups", [
    # one position: sixteen lanes a group; one channel a group; odd groups; one group; four vectors a lane; too wide for the registers
    ((37, 1024), 8), ((5, 16), 16), ((9, 1, 90), 6), ((3, 7), 1), ((1, 1024), 1), ((2, 2048), 1), ((2, 5000), 2), ((300, 48), 3), ((1, 1), 1),
    # many: ragged chunks, odd channels, one group of everything, a group wider than a workgroup's vectors, few positions
    ((2, 777, 180), 6), ((3, 130, 64), 4), ((1, 1000, 32), 1), ((2, 33, 3000), 1), ((2, 2, 8), 2), ((4, 9, 5, 24), 3), ((1, 3000, 7), 7),
    ((1, 64, 5120), 2),
], ids=str)
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_against_the_definition(shape, groups, dtype):
    for activation in (None, "silu", "gelu"):
        check(make(shape, dtype), groups, activation)


@pytest.mark.parametrize("params", [(True, False), (False, True), (False, False)], ids=str)
@pytest.mark.parametrize("shape", [(40, 64), (2, 100, 64)], ids=str)
def test_without_parameters(shape, params):
    check(make(shape, params=params), 4, "silu")


def test_parameters_in_another_type():
    x, weight, bias, up = make((2, 50, 64), BF16)
    want = run(definition, (x, weight, bias, up), 4, 1e-5, "silu", "cpu", torch.float64)
    for kinds in ((F32, F32), (BF16, F32)):
        got = run(hip_group_norm, (x, weight.to(kinds[0]), bias.to(kinds[1]), up), 4, 1e-5, "silu", "cuda")
        assert [g.dtype for g in got] == [BF16, BF16, *kinds]
        assert max(rel_err(g, w) for g, w in zip(got, want)) <= TOLERANCE[BF16]


@pytest.mark.parametrize("shape", [(8, 256), (2, 500, 64)], ids=str)
def test_values_far_from_zero(shape):
    """Means of 1000 beside deviations of 1: a value's own last place is 2^-14, which is what the result is off by."""
    check(make(shape, far=1000.0), 4, tolerance=2 ** -12)


def test_a_first_value_far_from_the_others():
    case = make((2, 300, 64))
    case[0][:, 0, 0] = 1e4
    check(case, 4)


def test_constant_groups_give_the_bias():
    x, weight, bias, up = make((3, 20, 32))
    x[1] = 2.5
    out = hip_group_norm(x.cuda(), 4, weight.cuda(), bias.cuda())
    assert torch.equal(out[1].cpu(), bias.expand(20, 32))


def test_views_are_read_as_they_are():
    x, weight, bias, up = make((2, 60, 96), BF16)
    part = torch.zeros(2, 60, 101, dtype=BF16)
    part[..., 3:99] = x
    want = run(hip_group_norm, (x, weight, bias, up), 4, 1e-5, "gelu", "cuda")
    leaf = part.cuda().requires_grad_(True)
    out = hip_group_norm(leaf[..., 3:99], 4, weight.cuda(), bias.cuda(), 1e-5, "gelu")
    (grad,) = torch.autograd.grad(out, leaf, up.cuda())
    assert torch.equal(out, want[0]) and torch.equal(grad[..., 3:99], want[1])
    assert rel_err(hip_group_norm(x.cuda().transpose(0, 1), 4), definition(x.double().transpose(0, 1), 4, None, None, 1e-5, None)) <= TOLERANCE[BF16]


def test_only_some_gradients_are_wanted():
    x, weight, bias, up = (t.cuda() for t in make((30, 64)))
    full = run(hip_group_norm, (x, weight, bias, up), 4, 1e-5, "silu", "cuda")
    weight.requires_grad_(True)
    (dw,) = torch.autograd.grad(hip_group_norm(x, 4, weight, bias, 1e-5, "silu"), weight, up)
    assert torch.equal(dw, full[2])
    (dx,) = torch.autograd.grad(hip_group_norm(x.requires_grad_(True), 4, None, bias, 1e-5, None), x, up)
    assert dx.shape == x.shape


def test_empty_batches():
    x = torch.zeros(0, 5, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    out = hip_group_norm(x, 4, w)
    assert out.shape == x.shape
    dx, dw = torch.autograd.grad(out.sum(), (x, w))
    assert dx.shape == x.shape and not dw.any()


def test_results_repeat_bit_for_bit():
    for shape in ((500, 256), (3, 700, 64)):
        case = make(shape, BF16)
        first, second = (run(hip_group_norm, case, 4, 1e-5, "silu", "cuda") for _ in range(2))
        assert all(torch.equal(a, b) for a, b in zip(first, second))


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_heads_of_a_recurrence(dtype):
    """The mixer as it is used: recurrence, a norm for each head, the output gate; forward and gradients."""
    from tests.test_hip_delta_gpu import make as delta_case, recurrence

    B, T, H, HV, K, V = 2, 100, 2, 4, 64, 48
    case = delta_case(B, T, H, HV, K, V, dtype=dtype, carried=False)
    x, weight, bias, up = make((B * T, HV * V), dtype)

    def mixer(q, k, v, g, b, w, c, gate, mixed, norm, output_gate):
        o = mixed(q, k, v, g, b)
        return output_gate(norm(o.reshape(B * T, HV * V), HV, w, c, 1e-5, None), gate)

    def leaves(device, kind=None):
        tensors = [case[n] for n in ("q", "k", "v", "log_decay", "beta")] + [weight, bias, x]
        return [t.to(device=device, dtype=kind or t.dtype).requires_grad_(True) for t in tensors]

    want_in, got_in = leaves("cpu", torch.float64), leaves("cuda")
    want = mixer(*want_in, lambda q, k, v, g, b: recurrence(q, k, v, g, b, None, K ** -0.5)[0], definition,
                 lambda h, v: h * F.gelu(v, approximate="tanh"))
    got = mixer(*got_in, lambda q, k, v, g, b: hip_gated_delta(q, k, v, g, b)[0], hip_group_norm, hip_gelu_gate)
    want_grads = torch.autograd.grad(want, want_in, up.double())
    got_grads = torch.autograd.grad(got, got_in, up.cuda())
    # three operators, each of which rounds what it hands on; the gradients come back through as many
    steps = 2 ** -8 if dtype == BF16 else 2 ** -16
    assert rel_err(got, want) <= 3 * steps
    for name, a, b in zip(("q", "k", "v", "log_decay", "beta", "weight", "bias", "gate"), got_grads, want_grads):
        assert rel_err(a, b) <= 6 * steps, name


@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", [(20, 64), (2, 70, 64)], ids=str)
def test_parameters_off_a_vector_boundary(shape, dtype):
    """... give what the same numbers on one give, bit for bit."""
    x, weight, bias, up = (t.cuda() for t in make(shape, dtype=dtype))
    results = []
    for offset in (0, 1):
        room = torch.zeros(2, shape[-1] + offset, dtype=dtype, device="cuda")
        room[0, offset:], room[1, offset:] = weight, bias
        leaves = [x.clone().requires_grad_(True), *(row[offset:].detach().requires_grad_(True) for row in room)]
        out = hip_group_norm(leaves[0], 4, leaves[1], leaves[2], activation="silu")
        results.append([out.detach(), *torch.autograd.grad(out, leaves, up)])
    assert all(torch.equal(a, b) for a, b in zip(*results))


def test_more_than_two_to_the_31_elements():
    """... whose offsets pass 32 bits: the last rows by themselves give the same."""
    rows, channels = (1 << 21) + 3, 1024
    x = torch.empty(rows, channels, dtype=BF16, device="cuda").normal_(generator=torch.Generator("cuda").manual_seed(1)).requires_grad_(True)
    out = hip_group_norm(x, 8)
    (grad,) = torch.autograd.grad(out, x, torch.ones((), dtype=BF16, device="cuda").expand_as(out) * out.detach())
    last = x.detach()[-64:].clone().requires_grad_(True)
    want = hip_group_norm(last, 8)
    (want_grad,) = torch.autograd.grad(want, last, want.detach())
    assert torch.equal(out[-64:], want) and torch.equal(grad[-64:], want_grad)


def test_sums_over_many_short_rows():
    """Gradients of the parameters over a million positions in rows of two.  A thread adds up 147 rows, a workgroup its lines and the last
    sum 2048 sets in 32 runs of 64: half a step of 2^-24 for each of fewer than 300 additions, all of them to one side for equal terms."""
    x, weight, bias, up = make((300000, 2, 8))
    up = torch.full_like(up, 1.1)
    got = run(hip_group_norm, (x, weight, bias, up), 2, 1e-5, None, "cuda")
    want = run(definition, (x, weight, bias, up), 2, 1e-5, None, "cpu", torch.float64)
    assert rel_err(got[3], want[3]) <= 2 ** -16, rel_err(got[3], want[3])
    # a weight's gradient cancels: its terms are 1.1 times xhat, of deviation 1
    assert float((got[2].cpu().double() - want[2]).abs().max()) <= 2 ** -16 * 1.1 * 600000
    assert rel_err(got[1], want[1]) <= 2 ** -12 and rel_err(got[0], want[0]) <= TOLERANCE[F32]
    case = make((40000, 3, 24), BF16)
    check(case, 3, "silu")


def test_more_rows_than_a_launch_holds():
    """2^24 rows of two positions: the ends and sums against the definition in 64 bits."""
    rows, C, groups = (1 << 24) + 3, 8, 2
    gen = torch.Generator("cuda").manual_seed(4)
    x, up = (torch.empty(rows, 2, C, dtype=BF16, device="cuda").normal_(generator=gen) for _ in range(2))
    weight, bias = (t.to(BF16).cuda() for t in make((2, C))[1:3])
    leaves = [t.requires_grad_(True) for t in (x, weight, bias)]
    out = hip_group_norm(x, groups, weight, bias, 1e-2, "silu")
    got = torch.autograd.grad(out, leaves, up)
    sums = [torch.zeros(C, dtype=torch.float64, device="cuda") for _ in range(2)]
    for at in range(0, rows, 1 << 20):
        part = [t[at : at + (1 << 20)].detach().double() if t.dim() == 3 else t.detach().double() for t in leaves]
        part = [t.requires_grad_(True) for t in part]
        want = definition(part[0], groups, *part[1:], 1e-2, "silu")
        grads = torch.autograd.grad(want, part, up[at : at + (1 << 20)].double())
        if at in (0, rows - rows % (1 << 20)):
            assert rel_err(out[at : at + (1 << 20)], want) <= TOLERANCE[BF16] and rel_err(got[0][at : at + (1 << 20)], grads[0]) <= TOLERANCE[BF16]
        for total, g in zip(sums, grads[1:]):
            total += g
    # terms of up to about 1 that cancel to their square root: 2^-16 of their number beside the rounding of the result
    for g, total in zip(got[1:], sums):
        assert ((g.double() - total).abs() <= 2 ** -8 * total.abs() + 2 ** -16 * 2 * rows).all()
