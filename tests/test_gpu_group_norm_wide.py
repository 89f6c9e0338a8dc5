"""nova_group_norm at sizes beyond the ordinary: more groups than a workgroup of
its layout's width has threads (three to seven channels a group above 2048
channels, channels-last), more elements than the element-by-element form's
grid, and what a training step keeps in memory. The definition in float64 and its
tolerances are test_gpu_group_norm.py's."""

import pytest
import torch

from test_gpu_group_norm import _case, _check

pytestmark = pytest.mark.gpu

SHAPES = [  # B, C, G, H, W
    (2, 2304, 768, 5, 5),     # forward in one launch
    (1, 2304, 768, 46, 47),   # forward in pieces
    (1, 2064, 688, 3, 7),
    (1, 4608, 768, 30, 21),
    (2, 5120, 1024, 9, 4),
    (1, 7168, 1024, 24, 25),
    (1, 8192, 1024, 5, 3),    # the most channels and groups
    (1, 2304, 576, 46, 47),   # as many groups as threads
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("shape", SHAPES)
def test_more_groups_than_threads(shape, dtype):
    B, C, G, H, W = shape
    print(f"[group norm] {shape} {dtype}", flush=True)
    x, w, b, gy = _case(B, C, H, W, dtype, True, seed=C)
    _check(x, G, w, b, gy, silu=C % 5 != 0)


def test_more_elements_than_the_plain_grid():
    """Two images of 2^27 elements and more each: the element-by-element form's
    gradient walks further than its grid, and gives each image what it gives it
    alone."""
    from nova_winograd import nova_group_norm

    C, H, W = 16384, 82, 100
    g = torch.Generator(device="cuda").manual_seed(1)
    x, gy = (torch.randn(2, H, W, C, generator=g, device="cuda", dtype=torch.float16)
             .permute(0, 3, 1, 2) for _ in "xg")
    both = x.detach().requires_grad_()
    nova_group_norm(both, 32, activation="silu").backward(gy)
    for i in range(2):
        one = x[i:i + 1].detach().requires_grad_()
        nova_group_norm(one, 32, activation="silu").backward(gy[i:i + 1])
        assert torch.equal(one.grad, both.grad[i:i + 1])
        assert one.grad.count_nonzero() > 0.9 * one.numel()


@pytest.mark.parametrize("shape", [(4, 10240, 32, 3, 3), (4, 320, 32, 64, 64), (64, 960, 32, 5, 3)])
@pytest.mark.parametrize("nhwc", [True, False])
def test_memory_kept_for_the_backward(shape, nhwc):
    """The statistics, 8 bytes for each image and group, and of the workspace at
    most 1/16 of the input."""
    from nova_winograd import nova_group_norm

    B, C, G, H, W = shape
    x = _case(B, C, H, W, torch.float16, nhwc)[0].requires_grad_()
    nova_group_norm(x, G)
    before = torch.cuda.memory_allocated()
    y = nova_group_norm(x, G)
    kept = torch.cuda.memory_allocated() - before - 2 * y.numel()
    assert kept <= 8 * B * G + x.numel() // 8 + 2 * 512  # the allocator's blocks
