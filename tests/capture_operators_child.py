"""Graph captures of the gated delta rule and the group norm for test_hip_delta_gpu, in a process of their own.  Prints a line for each
case, ends with status 1 after a mismatch."""

import sys

import torch

from griffin_amd import hip_gated_delta, hip_gated_delta_step, hip_group_norm

BF16, F32 = torch.bfloat16, torch.float32


def tensors(*shapes, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(*shape, generator=gen).to(dtype).cuda() for shape in shapes]


def delta(dtype, B, T, H, HV, K, V, masked):
    q, k, v, decay, beta = tensors((B, T, H, K), (B, T, H, K), (B, T, HV, V), (B, T, HV), (B, T, HV), dtype=dtype, seed=1)
    leaves = [torch.nn.functional.normalize(q, dim=-1), torch.nn.functional.normalize(k, dim=-1), v, -torch.nn.functional.softplus(decay - 3), beta.sigmoid()]
    active = torch.arange(T, device="cuda")[None] < torch.tensor([[T], [T // 2]], device="cuda")[:B] if masked else None
    reset = torch.arange(T, device="cuda")[None].expand(B, T) % 50 == 0 if masked else None
    return leaves, lambda *x: hip_gated_delta(*x, reset_mask=reset, active_mask=active)


def heads(dtype, *shape):
    x, w, b = tensors(shape, shape[-1:], shape[-1:], dtype=dtype, seed=2)
    return [x, w, b], lambda *t: (hip_group_norm(t[0], 4, t[1], t[2], activation="silu"),)


CASES = [
    ("delta", delta, (F32, 2, 150, 2, 2, 64, 48, False)),
    ("delta, masked, shared keys, odd rows", delta, (BF16, 2, 150, 1, 2, 50, 20, True)),
    ("delta in segments", delta, (BF16, 1, 1200, 1, 1, 128, 64, True)),
    ("norm of heads", heads, (BF16, 70, 64)),
    ("norm over positions", heads, (F32, 2, 300, 64)),
]


def whole_pass(make, args):
    """Forward and backward in one graph, replayed with new contents between eager calls: bit for bit the eager results."""
    leaves, forward = make(*args)
    leaves = [t.requires_grad_(True) for t in leaves]
    ups = [torch.randn_like(t) for t in forward(*leaves)]
    gradients = lambda: (lambda outs: [*(o.detach() for o in outs), *torch.autograd.grad(outs, leaves, ups)])(forward(*leaves))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            gradients()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = gradients()
    good = True
    for i in range(4):
        with torch.no_grad():
            leaves[0].copy_(leaves[0].roll(1, 0).neg())
            leaves[2].mul_(0.5)
            ups[0].copy_(ups[0].flip(0))
        want = [t.clone() for t in gradients()]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        good &= all(torch.equal(a, b) for a, b in zip(got, want))
    return good


def backward_alone(make, args):
    """The backward pass over an eager forward, captured and replayed for several upstream gradients."""
    leaves, forward = make(*args)
    leaves = [t.requires_grad_(True) for t in leaves]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        outs = forward(*leaves)
        choices = [[torch.randn_like(t) for t in outs] for _ in range(3)]
        want = [[g.clone() for g in torch.autograd.grad(outs, leaves, up, retain_graph=True)] for up in choices]
        ups = [t.clone() for t in choices[0]]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = torch.autograd.grad(outs, leaves, ups, retain_graph=True)
    good = True
    for choice, expected in zip(choices, want):
        for a, b in zip(ups, choice):
            a.copy_(b)
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        good &= all(torch.equal(a, b) for a, b in zip(got, expected))
    return good


def steps():
    """Two graphs of single tokens, captured one after the other and replayed in turn, each on a state of its own."""
    good, graphs = True, []
    for dtype in (F32, BF16):
        (q, k, v, decay, beta), state = tensors((3, 2, 64), (3, 2, 64), (3, 2, 40), (3, 2), (3, 2), dtype=dtype, seed=4), torch.zeros(3, 2, 64, 40, device="cuda")
        decay = -decay.abs()
        flags = torch.tensor([0, 2, 1], dtype=torch.uint8, device="cuda")
        token = lambda s, q=q, k=k, v=v, decay=decay, beta=beta, flags=flags: hip_gated_delta_step(q, k, v, decay, beta, s, flags=flags)
        token(state.clone())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = token(state)
        graphs.append((graph, token, state, out, state.clone(), v))
    for i in range(4):
        for graph, token, state, out, eager, v in graphs:
            v.mul_(1.25)
            want = token(eager)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            good &= torch.equal(out, want) and torch.equal(state, eager)
    return good


def main():
    good = True
    for name, make, args in CASES:
        for what in (whole_pass, backward_alone):
            print(what.__name__, name, flush=True)
            ok = what(make, args)
            print("  ", "equal" if ok else "DIFFERENT", flush=True)
            good &= ok
    print("steps", flush=True)
    ok = steps()
    print("  ", "equal" if ok else "DIFFERENT", flush=True)
    return good and ok


if __name__ == "__main__":
    sys.exit(0 if main() else 1)
