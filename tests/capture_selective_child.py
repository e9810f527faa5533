"""Graph captures of the selective scan, its convolution and the norm with the residual's addition for test_hip_selective_gpu, in a process of their
own.  Prints a line for each case, ends with status 1 after a mismatch."""

import sys

import torch

from griffin_amd import (hip_add_rmsnorm, hip_add_rmsnorm_quantised, hip_selective_scan, hip_selective_step, hip_short_conv,
                         hip_short_conv_step)

BF16, F32 = torch.bfloat16, torch.float32


def tensors(*shapes, dtype, seed):
    gen = torch.Generator().manual_seed(seed)
    return [torch.randn(*shape, generator=gen).to(dtype).cuda() for shape in shapes]


def masks(B, T):
    active = torch.arange(T, device="cuda")[None] < torch.tensor([[T], [T // 2]], device="cuda")[:B]
    return torch.arange(T, device="cuda")[None].expand(B, T) % 50 == 0, active


def scan(dtype, B, T, W, G, N, masked):
    u, dt, b, c, z = tensors((B, T, W), (B, T, W), (B, T, G, N), (B, T, G, N), (B, T, W), dtype=dtype, seed=1)
    A, D, h0 = tensors((W, N), (W,), (B, W, N), dtype=F32, seed=2)
    reset, active = masks(B, T) if masked else (None, None)
    return [u, dt, -A.abs(), b, c, D, z, D * 0.1 - 2, h0], lambda *x: hip_selective_scan(*x, reset_mask=reset, active_mask=active)


def conv(dtype, B, T, W, K, masked):
    leaves = tensors((B, T, W), (W, 1, K), (W,), (B, K - 1, W), dtype=dtype, seed=3)
    reset, active = masks(B, T) if masked else (None, None)
    return leaves, lambda *x: hip_short_conv(*x, "silu", reset, active, need_state=False)[:1]


def norm(dtype, residual, *shape):
    return [*tensors(shape, dtype=dtype, seed=4), *tensors(shape, dtype=residual, seed=5), *tensors(shape[-1:], dtype=dtype, seed=6)], hip_add_rmsnorm


CASES = [
    ("scan", scan, (F32, 2, 150, 40, 1, 16, False)),
    ("scan, masked, groups, odd states", scan, (BF16, 2, 150, 36, 2, 13, True)),
    ("scan in segments", scan, (BF16, 1, 1200, 20, 1, 16, True)),
    ("scan of many states", scan, (F32, 2, 70, 20, 1, 40, False)),
    ("convolution", conv, (BF16, 2, 150, 64, 4, False)),
    ("convolution, masked", conv, (F32, 2, 150, 33, 4, True)),
    ("norm", norm, (BF16, F32, 70, 64)),
    ("wide norm", norm, (F32, F32, 30, 2000)),
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
            leaves[1].mul_(0.5)
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
    """Two graphs of single tokens, captured one after the other and replayed in turn, each on states of its own."""
    good, graphs = True, []
    for dtype in (F32, BF16):
        x, dt, b, c, z, weight, bias, window = tensors((3, 40), (3, 40), (3, 2, 16), (3, 2, 16), (3, 40), (40, 1, 4), (40,), (3, 3, 40), dtype=dtype, seed=7)
        A, D, state, g = tensors((40, 16), (40,), (3, 40, 16), (40,), dtype=F32, seed=8)
        A, flags = -A.abs(), torch.tensor([0, 2, 1], dtype=torch.uint8, device="cuda")

        def token(window, state, x=x, dt=dt, b=b, c=c, z=z, weight=weight, bias=bias, A=A, D=D, g=g, flags=flags):
            u = hip_short_conv_step(x, weight, bias, window, "silu", flags)
            y = hip_selective_step(u, dt, A, b, c, state, D, z, flags=flags)
            q, scale, _ = hip_add_rmsnorm_quantised(y, None, g)
            return [u, y, q.float(), scale]

        token(window.clone(), state.clone())
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = token(window, state)
        graphs.append((graph, token, (window, state), out, (window.clone(), state.clone()), x))
    for i in range(4):
        for graph, token, held, out, eager, x in graphs:
            x.mul_(1.25)
            want = token(*eager)
            torch.cuda.synchronize()
            graph.replay()
            torch.cuda.synchronize()
            good &= all(torch.equal(a, b) for a, b in zip([*out, *held], [*want, *eager]))
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
