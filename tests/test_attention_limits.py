"""The launch limits of attention's C entry points, both sides of each, on the
CPU (argument checks alone: a grid holds fewer than 2^32 threads, and every
head of a sequence takes a workgroup of 256)."""

import pytest


def _args(**kw):
    from nova_winograd.ops import AttentionArgs, Strides

    a = AttentionArgs()
    a.q = a.k = a.v = 16
    a.q_strides = a.k_strides = a.v_strides = Strides(8, 8, 8)
    a.dtype, a.batch, a.kv_batch, a.queries, a.keys = 0, 1, 1, 1, 1
    a.heads, a.kv_heads, a.head_dim, a.scale = 1, 1, 8, 0.25
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("fits,over", [
    (dict(batch=2 ** 24 - 1, kv_batch=1), dict(batch=2 ** 24, kv_batch=1)),
    (dict(batch=2 ** 24 - 1, kv_batch=1, queries=3, keys=200),
     dict(batch=2 ** 24, kv_batch=1, queries=3, keys=200)),
    (dict(batch=2 ** 20, kv_batch=1, heads=15), dict(batch=2 ** 20, kv_batch=1, heads=16)),
    (dict(batch=0, heads=2 ** 24 - 1, kv_heads=2 ** 24 - 1),
     dict(batch=0, heads=2 ** 24, kv_heads=2 ** 24)),
    (dict(queries=2 ** 28), dict(queries=2 ** 28 + 1)),
    (dict(keys=2 ** 28), dict(keys=2 ** 28 + 1)),
    (dict(batch=2 ** 9, kv_batch=1, queries=2 ** 20),
     dict(batch=2 ** 9 + 1, kv_batch=1, queries=2 ** 20)),
])
def test_launch_limits(fits, over):
    from nova_winograd.ops import get_lib

    lib = get_lib()
    lib.nova_get_last_error()
    for backward in (0, 1):
        assert lib.nova_cross_attention_workspace_bytes(_args(**fits), backward) >= 0
        assert lib.nova_get_last_error() == 0
        assert lib.nova_cross_attention_workspace_bytes(_args(**over), backward) == -1
        assert lib.nova_get_last_error() == 1
    lib.nova_cross_attention(_args(**over), 16, None, None, None, 0, None)
    assert lib.nova_get_last_error() == 1
    lib.nova_cross_attention_backward(_args(**over), 16, 16, 16, 16, 16, 16, 16, None, 0, None)
    assert lib.nova_get_last_error() == 1
