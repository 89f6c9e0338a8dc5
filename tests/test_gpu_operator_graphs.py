"""Whole training steps of nova_group_norm and nova_cross_attention in a graph:
every replay gives the eager step's bits, with eager steps between them."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def _replays(step, leaves):
    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    originals = [t.detach().clone() for t in leaves]
    for i in range(4):
        with torch.no_grad():  # other inputs and back: a replay reads them anew
            for t, o in zip(leaves, originals):
                t.copy_(o * (0.5 if i == 1 else 1.0))
        for t in got:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        eager = step()
        assert all(torch.equal(a, b) for a, b in zip(got, eager)), i
        assert i == 1 or all(torch.equal(a, b) for a, b in zip(got, want)), i


@pytest.mark.parametrize("shape", [  # B, Lq, Lk, H, KV, D
    (4, 512, 77, 8, 8, 40),     # one workgroup holds the keys; sums joined
    (3, 500, 333, 4, 2, 80),    # tiles
    (1, 30, 1500, 4, 4, 64),    # few rows, keys split
    (4, 1, 1500, 8, 2, 64),     # one token
    (2, 256, 600, 64, 64, 128),  # two groups of waves
])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_attention_step(shape, dtype):
    import nova_winograd as nw

    B, Lq, Lk, H, KV, D = shape
    print(f"[attention graph] {shape} {dtype}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(D)
    leaves = [torch.randn(B, n, h, D, generator=g, device=DEV).to(dtype).requires_grad_()
              for n, h in ((Lq, H), (Lk, KV), (Lk, KV))]
    go = torch.randn(B, Lq, H, D, generator=g, device=DEV).to(dtype)
    mask = torch.rand(B, Lk, generator=g, device=DEV) < 0.8

    def step():
        out = nw.nova_cross_attention(*leaves, mask)
        return (out.detach(), *torch.autograd.grad(out, leaves, go))

    _replays(step, leaves)


@pytest.mark.parametrize("nhwc", [True, False])
@pytest.mark.parametrize("shape", [(2, 320, 32, 64, 64), (1, 1280, 32, 8, 8), (3, 30, 5, 31, 17),
                                   (1, 2304, 768, 9, 9), (2, 1031, 1, 5, 5)])
def test_group_norm_step(shape, nhwc):
    import nova_winograd as nw

    B, C, G, H, W = shape
    print(f"[group norm graph] {shape} nhwc={nhwc}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(C)
    fmt = torch.channels_last if nhwc else torch.contiguous_format
    x, gy = (torch.randn(B, C, H, W, generator=g, device=DEV).half().contiguous(memory_format=fmt)
             for _ in "xg")
    leaves = [x.requires_grad_()] + [torch.randn(C, generator=g, device=DEV).requires_grad_()
                                     for _ in "wb"]

    def step():
        y = nw.nova_group_norm(leaves[0], G, leaves[1], leaves[2], activation="silu")
        return (y.detach(), *torch.autograd.grad(y, leaves, gy))

    _replays(step, leaves)
