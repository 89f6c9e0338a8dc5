"""Host rules of group norm's launches, on the CPU: workgroups that a launch
takes for every number of channels and groups, and the C entry points' launch
limits, both sides of each."""

import pytest

from host_program import build

PROGRAM = """
#include <cstdio>
#include "nova_internal.h"
int main() {
    int dtype, B, C, G, nhwc, backward;
    long long P;
    while (std::scanf("%d %d %d %d %lld %d %d", &dtype, &B, &C, &G, &P, &nhwc, &backward) == 7) {
        nova::GroupNorm g{};
        g.dtype = dtype;
        g.B = B;
        g.C = C;
        g.G = G;
        g.P = P;
        g.nhwc = nhwc;
        const nova::GroupNormLaunch l = nova::group_norm_launch(g, backward != 0, 256);
        std::printf("%lld %d\\n", (long long)l.threads, l.block);
    }
}
"""


@pytest.fixture(scope="module")
def launches(tmp_path_factory):
    return build(tmp_path_factory.mktemp("group_norm_plan"), PROGRAM)


def test_workgroups_for_every_width(launches):
    rows = []
    for C in [*range(1, 400, 7), *range(400, 9300, 24), 1032, 2054, 2304, 7168, 8192]:
        for n in (1, 2, 3, 4, 5, 6, 7, 8, 10, 32, C):
            if C % n == 0:
                rows += [(t, 2, C, C // n, P, nhwc, bwd) for t in (0, 2) for P in (25, 3000)
                         for nhwc in (0, 1) for bwd in (0, 1)]
    for row, (_, block) in zip(rows, launches(rows)):
        assert 64 <= block <= 1024 and block % 64 == 0, row


def _args(**kw):
    from nova_winograd.ops import GroupNormArgs

    a = GroupNormArgs(16, None, None, 0, 2, 1, 1, 1, 0, 1, 1e-5, 1)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


LIMITS = [  # the largest batch (or number of pixels) that fits, forward and backward
    # a workgroup of 256 threads for every image and group: 2^24 of them
    ("batch", 524287, 524287, dict(channels=256, groups=32)),
    ("batch", 524287, 524287, dict(channels=256, groups=32, channels_last=1)),
    ("batch", 16777215, 16777215, dict()),
    # 64 threads for every image and channel
    ("batch", 1048575, 1048575, dict(channels=64, groups=1, pixels=1000)),
    # more groups than 1024, or channels than 1024 vectors: a workgroup for every
    # image and group, and in the backward for every channel too
    ("batch", 8191, 8191, dict(channels=2048, groups=2048, channels_last=1)),
    # (forward: 2^30 images times channels)
    ("batch", 65536, 1023, dict(channels=16384, groups=32, channels_last=1)),
    # the walk over the pixels
    ("pixels", 2 ** 31 - 1 - 2 ** 20, 2 ** 31 - 1 - 2 ** 20, dict()),
    ("pixels", 2 ** 31 - 1 - 2 ** 20, 2 ** 31 - 1 - 2 ** 20, dict(channels=8, channels_last=1)),
]


@pytest.mark.parametrize("name,forward,backward,rest", LIMITS)
def test_launch_limits(name, forward, backward, rest):
    from nova_winograd.ops import get_lib

    lib = get_lib()
    lib.nova_get_last_error()
    for bwd, most in ((0, forward), (1, backward)):
        assert lib.nova_group_norm_workspace_bytes(_args(**rest, **{name: most}), bwd) >= 0
        assert lib.nova_get_last_error() == 0
        over = _args(**rest, **{name: most + 1})
        assert lib.nova_group_norm_workspace_bytes(over, bwd) == -1
        assert lib.nova_get_last_error() == 1
        if bwd:
            lib.nova_group_norm_backward(over, 16, 16, 16, 16, 16, 16, 16, 1 << 50, None)
        else:
            lib.nova_group_norm(over, 16, 16, 16, 16, 1 << 50, None)
        assert lib.nova_get_last_error() == 1
        assert b"launch limits" in lib.nova_get_last_error_message()


def test_tensors_past_2_pow_32_elements_are_taken(launches):
    # the plain form's walk over 2^33 elements
    for bwd in (0, 1):
        assert _fits(launches, (0, 1, 16384, 32, 2 ** 19, 1, bwd))


def _fits(launches, row):
    (threads, block), = launches([row])
    return threads < 2 ** 32 and block <= 1024
