"""nova_cross_attention where it can go wrong beside its ordinary range: rows
whose scores leave nothing at any scale, and rows whose output gradients lie far
apart. The definition in float64 and its tolerances are test_gpu_attention.py's
where nothing else is said."""

import pytest
import torch

from test_gpu_attention import DEV, _compare, _nw, _randn, _run

pytestmark = pytest.mark.gpu


EMPTY = [  # B, Lq, Lk, H, KV, D
    (3, 1, 77, 4, 2, 40),       # few rows
    (3, 2, 300, 4, 4, 64),      # few rows, keys split over workgroups
    (3, 5, 77, 4, 2, 40),       # all keys in one workgroup, gradients over tiles
    (3, 200, 60, 4, 2, 40),     # ... and the gradients by one workgroup too
    (3, 200, 77, 4, 4, 64),
    (3, 200, 128, 2, 2, 160),
    (3, 200, 129, 4, 2, 40),    # tiles of keys
    (4, 256, 130, 32, 32, 128),  # two groups of waves
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scale", [0.0, -0.3, 0.69, 0.7, 1.0, -1.0, 1.5])
@pytest.mark.parametrize("shape", EMPTY)
def test_rows_without_keys_at_any_scale(shape, scale, dtype):
    """Zeros and no gradient, whatever the scale."""
    B, Lq, Lk, H, KV, D = shape
    print(f"[attention] {shape} {scale} {dtype}", flush=True)
    g = torch.Generator(device=DEV).manual_seed(D + Lk)
    q = _randn(g, B, Lq, H, D, dtype=dtype)
    k, v = _randn(g, B, Lk, KV, D, dtype=dtype), _randn(g, B, Lk, KV, D, dtype=dtype)
    mask = torch.rand(B, Lk, generator=g, device=DEV) < 0.5
    mask[:, Lk - 1] = True
    mask[1] = False
    # scores of a standard deviation of about 1
    _run((q.float() / D ** 0.5).to(dtype), k, v, mask, scale=scale)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = _nw().nova_cross_attention(*leaves, mask, scale)
    out.backward(torch.ones_like(out))
    assert not out[1].any() and out.isfinite().all()
    for t in leaves:
        assert not t.grad[1].any() and t.grad.isfinite().all()


@pytest.mark.parametrize("Lq", [1, 5, 200])
@pytest.mark.parametrize("D", [1, 2])
def test_rows_without_keys_at_the_default_scale(Lq, D):
    """One and two channels, whose default scale is above ln 2."""
    g = torch.Generator(device=DEV).manual_seed(D)
    q, k, v = (_randn(g, 4, n, 2, D) for n in (Lq, 50, 50))
    mask = torch.rand(4, 50, generator=g, device=DEV) < 0.7
    mask[2] = False
    assert not _run(q, k, v, mask)[2].any()


@pytest.mark.parametrize("scale", [0.3, 2.0])
@pytest.mark.parametrize("Lq,Lk,H,D", [(1, 300, 2, 8), (40, 100, 2, 8), (40, 300, 2, 8),
                                       (256, 300, 32, 128)])
def test_scores_of_minus_infinity(Lq, Lk, H, D, scale):
    """Kept keys whose scores are -inf take no part, a whole tile of them in
    front included; a row that has only such keys gives zeros."""
    nw = _nw()
    g = torch.Generator(device=DEV).manual_seed(3)
    B = 4
    q = _randn(g, B, Lq, H, D, dtype=torch.bfloat16).abs() + 0.25
    k, v = (_randn(g, B, Lk, H, D, dtype=torch.bfloat16) for _ in "kv")
    out_of = torch.zeros(B, Lk, dtype=torch.bool, device=DEV)
    out_of[0, :70] = True
    out_of[1] = torch.rand(Lk, generator=g, device=DEV) < 0.5
    out_of[2] = True
    dead = k.clone()
    dead[..., 0] = torch.where(out_of[:, :, None], float("-inf"), k[..., 0])
    with torch.no_grad():
        got = nw.nova_cross_attention(q, dead, v, scale=scale)
        want = nw.nova_cross_attention(q, k, v, ~out_of, scale)
    assert not got[2].any()
    # the walk over tiles may take the kept keys in other steps: one rounding
    # of p and one of the output on each side
    size = v.abs().amax(dim=(1, 3)).view(B, 1, H, 1).double()
    tol = 4 * 2.0 ** -8 * size.expand_as(got)
    _compare([got], [(want.double(), tol)], ["out"])


def _query_gradient(q, k, v, go):
    """float64, without a mask: grad_q and a bound on its error that holds each
    row to its own values. ds is rounded to float16 (u), at a power of two that
    leaves it off by 2^-32 of the row's largest where it is small; its float32
    parts (see test_gpu_attention.py) are off by e; delta is their sum."""
    D = q.shape[3]
    u, e = 2.0 ** -11, 2.0 ** -24
    Q, K, V, G = (t.double().transpose(1, 2).contiguous() for t in (q, k, v, go))
    kt, vt = K.transpose(2, 3).contiguous(), V.transpose(2, 3).contiguous()
    p = torch.softmax(torch.matmul(Q, kt) * D ** -0.5, 3)
    top = (torch.matmul(Q.abs(), kt.abs()) * D ** -0.5).amax(3, keepdim=True)
    rel = u + 4 * (D + 4) * e * top + 2.0 ** -19
    dp, size = torch.matmul(G, vt), torch.matmul(G.abs(), vt.abs())
    ds = p * (dp - (p * dp).sum(3, keepdim=True))
    off = ds.abs() * rel + 2.0 ** -31 * ds.abs().amax(3, keepdim=True)
    off = off + p * (D + 4) * e * (size + 2 * size.amax(3, keepdim=True))
    dq = torch.matmul(ds, K) * D ** -0.5
    tol = torch.matmul(off, K.abs()) * D ** -0.5 + u * dq.abs() + 2.0 ** -24
    return dq.transpose(1, 2), tol.transpose(1, 2)


@pytest.mark.parametrize("Lk,D", [(20, 64), (60, 40), (77, 40), (77, 64), (96, 160), (128, 80),
                                  (129, 64)])
def test_rows_with_gradients_far_apart(Lk, D):
    """Each row's grad_q keeps the type's precision beside rows whose gradients
    are 2^20 times as large, and beside rows that have none (float16)."""
    g = torch.Generator(device=DEV).manual_seed(Lk)
    B, H, Lq = 2, 2, 300
    q, k, v = (_randn(g, B, n, H, D) for n in (Lq, Lk, Lk))
    go = torch.randn(B, Lq, H, D, generator=g, device=DEV)
    go[:, 2::3] = 0.0
    for high, low in ((2.0 ** 10, 2.0 ** -10), (2.0 ** -4, 2.0 ** -4), (2.0 ** -20, 2.0 ** -20)):
        gr = go.clone()
        gr[:, ::3] *= high
        gr[:, 1::3] *= low
        gr = gr.half()
        leaves = [t.clone().requires_grad_() for t in (q, k, v)]
        _nw().nova_cross_attention(*leaves).backward(gr)
        _compare([leaves[0].grad], [_query_gradient(q, k, v, gr)], ["grad_q"])
        assert not leaves[0].grad[:, 2::3].any()
        assert all(t.grad.isfinite().all() for t in leaves)
