"""Arguments of nova_group_norm and nova_cross_attention that the C structures
behind them cannot hold."""

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
