"""Arguments of nova_group_norm and nova_cross_attention that they have to
refuse: sizes that the C structures behind them cannot hold, and tensors with a
forward-mode tangent."""

import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = torch.device("cuda:0")


def test_sizes_past_32_bits_are_refused():
    """2^32 + 2 must not be taken for 2. The tensors repeat one value."""
    import nova_winograd as nw

    many = 2 ** 32 + 2
    one = torch.ones(1, 1, 1, 1, device=DEV, dtype=torch.float16)
    for shape in ((many, 1, 1, 1), (1, many, 1, 1)):
        with pytest.raises(ValueError, match="launch limits"):
            nw.nova_group_norm(one.expand(shape), 1)
    for shape in ((1, 1, 1, many), (1, 1, many, 1)):  # as pixels: the C entry's own limit
        with pytest.raises(RuntimeError, match="launch limits"):
            nw.nova_group_norm(torch.empty(0, 1, 1, 1, device=DEV).expand(0, *shape[1:]), 1)
    small = one.expand(1, 2, 1, 8)
    for q, k in ((one.expand(many, 1, 1, 8), small), (one.expand(1, many, 1, 8), small),
                 (one.expand(1, 1, many, 8), small), (small, one.expand(1, many, 1, 8)),
                 (one.expand(1, 1, 1, many), one.expand(1, 1, 1, many))):
        with pytest.raises(ValueError, match="launch limits"):
            nw.nova_cross_attention(q, k, k)


@pytest.mark.parametrize("requires_grad", [False, True])
@pytest.mark.parametrize("grad_mode", [False, True])
def test_forward_mode_is_refused(requires_grad, grad_mode):
    """A tangent is not dropped in silence, whichever input brings it."""
    import nova_winograd as nw
    import torch.autograd.forward_ad as fw

    def rand(*s, dtype=torch.float16):
        return torch.randn(*s, device=DEV, dtype=dtype).requires_grad_(requires_grad)

    norm = [rand(2, 8, 3, 3), rand(8, dtype=torch.float32), rand(8, dtype=torch.float32)]
    attention = [rand(2, 5, 2, 16), rand(2, 7, 2, 16), rand(2, 7, 2, 16)]
    with torch.set_grad_enabled(grad_mode), fw.dual_level():
        for i in range(3):
            dual = list(norm)
            dual[i] = fw.make_dual(norm[i], torch.ones_like(norm[i]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                nw.nova_group_norm(dual[0], 4, dual[1], dual[2])
            dual = list(attention)
            dual[i] = fw.make_dual(attention[i], torch.ones_like(attention[i]))
            with pytest.raises(NotImplementedError, match="forward-mode"):
                nw.nova_cross_attention(*dual)
        # inside a dual level, without a tangent, nothing changes
        assert nw.nova_group_norm(norm[0], 4).requires_grad == (requires_grad and grad_mode)
        assert nw.nova_cross_attention(*attention).requires_grad == (requires_grad and grad_mode)
