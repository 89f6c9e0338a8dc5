"""nova_cross_attention where it can go wrong beside its ordinary range: rows
whose scores leave nothing at any scale, rows whose output gradients lie far
apart, and what the gradients keep beyond one rounding of p, ds and the output. The definition in float64 and its tolerances are test_gpu_attention.py's
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


@pytest.mark.parametrize("shape,dtype", [  # B, Lq, Lk, H, KV, D
    ((1, 1, 64, 1, 1, 64), torch.bfloat16),
    ((1, 1, 1, 1, 1, 40), torch.bfloat16),
    ((2, 33, 50, 4, 2, 40), torch.bfloat16),
    ((1, 512, 64, 1, 1, 64), torch.bfloat16),
    ((8, 1, 20, 8, 2, 160), torch.bfloat16),
    ((1, 64, 33, 2, 1, 256), torch.bfloat16),
    ((1, 100, 64, 2, 2, 8), torch.float16),
    ((4, 16, 40, 8, 8, 4), torch.float16),
])
def test_two_terms_for_few_rows(shape, dtype):
    """Up to 512 rows in a call p and ds enter the gradients' products as two
    terms each: a rounding of u^2 in place of u. (Up to 64 keys, where delta is a
    sum in float32. The types and sizes are those at which u is far above
    float32's own errors in a score.)"""
    B, Lq, Lk, H, KV, D = shape
    u, e = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype], 2.0 ** -24
    tiny = 2.0 ** -24 if dtype is torch.float16 else 1e-38
    g = torch.Generator(device=DEV).manual_seed(Lk + D)
    q, go = (_randn(g, B, Lq, H, D, dtype=dtype) for _ in "qg")
    k, v = (_randn(g, B, Lk, KV, D, dtype=dtype) for _ in "kv")
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    _nw().nova_cross_attention(*leaves).backward(go)

    def heads(t):
        return t.double().transpose(1, 2).repeat_interleave(H // t.shape[2], 1).contiguous()

    def fold(t):
        return t.view(B, KV, H // KV, Lk, D).sum(2).transpose(1, 2)

    def turned(t):
        return t.transpose(2, 3).contiguous()

    Q, K, V, G = heads(q), heads(k), heads(v), heads(go)
    scale = D ** -0.5
    p = torch.softmax(torch.matmul(Q, turned(K)) * scale, 3)
    top = (torch.matmul(Q.abs(), turned(K).abs()) * scale).amax(3, keepdim=True)
    rel = 4 * u * u + 4 * (D + 4) * e * top + 2.0 ** -19
    dp, size = torch.matmul(G, turned(V)), torch.matmul(G.abs(), turned(V).abs())
    ds = p * (dp - (p * dp).sum(3, keepdim=True))
    off = ds.abs() * rel + p * (D + 4) * e * (size + 2 * size.amax(3, keepdim=True))
    # float16: what is left of a row's (a key's) small values
    row, key = (2.0 ** -31 * ds.abs().amax(d, keepdim=True) for d in (3, 2))
    dq = torch.matmul(ds, K) * scale
    dq_tol = torch.matmul(off + row, K.abs()) * scale
    dk = fold(torch.matmul(turned(ds), Q) * scale)
    dk_tol = fold(torch.matmul(turned(off + key), Q.abs()) * scale)
    dv = fold(torch.matmul(turned(p), G))
    dv_tol = fold(torch.matmul(turned(p * rel + 2.0 ** -34), G.abs()))
    want = [(dq.transpose(1, 2), dq_tol.transpose(1, 2)), (dk, dk_tol), (dv, dv_tol)]
    _compare([t.grad for t in leaves], [(x, t + u * x.abs() + tiny) for x, t in want],
             ["grad_q", "grad_k", "grad_v"])


def _rounded_terms(q, k, v, go, u, rest):
    """float64: grad_q, and the 2-norms that its error's independent parts have
    at most, as an array: ds rounded, the forward's p rounded (through delta =
    do . o), grad_q rounded, and without rest o rounded (through delta too)."""
    D = q.shape[3]
    Q, K, V, G = (t.double().transpose(1, 2).contiguous() for t in (q, k, v, go))
    kt, vt = K.transpose(2, 3).contiguous(), V.transpose(2, 3).contiguous()
    p = torch.softmax(torch.matmul(Q, kt) * D ** -0.5, 3)
    dp, o = torch.matmul(G, vt), torch.matmul(p, V)
    ds = p * (dp - (G * o).sum(3, keepdim=True))
    dq, pk = torch.matmul(ds, K) * D ** -0.5, torch.matmul(p, K) * D ** -0.5
    parts = [(torch.matmul(ds ** 2, K ** 2) / D).sum(),
             ((p ** 2 * dp ** 2).sum(3, keepdim=True) * pk ** 2).sum(), (dq ** 2).sum()]
    if not rest:
        parts.append(((G ** 2 * o ** 2).sum(3, keepdim=True) * pk ** 2).sum())
    return dq.transpose(1, 2), u * torch.stack(parts).sum().sqrt().item()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("Lq,Lk", [(700, 1000), (700, 333), (40, 1000)])
def test_rest_of_the_output(dtype, Lq, Lk):
    """Over tiles of keys delta comes from the output and what its rounding
    dropped. Keys and values with a common part far above their spread make
    grad_q feel delta's error; without rest it is several times the bound of the
    other roundings, and below the bound that takes the output's in."""
    from nova_winograd.ops import AttentionArgs, Strides, get_lib

    B, H, D = 1, 1, 64
    u = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}[dtype]
    g = torch.Generator(device=DEV).manual_seed(Lk)
    q = (0.25 * torch.randn(B, Lq, H, D, generator=g, device=DEV)).to(dtype)
    k, v = ((4 + torch.randn(B, Lk, H, D, generator=g, device=DEV)).to(dtype) for _ in "kv")
    go = _randn(g, B, Lq, H, D, dtype=dtype)
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = _nw().nova_cross_attention(*leaves)
    out.backward(go)
    dq, bound = _rounded_terms(q, k, v, go, u, True)
    assert (leaves[0].grad.double() - dq).norm().item() <= bound

    # the C entry points, rest not given
    a = AttentionArgs()
    a.q, a.k, a.v = q.data_ptr(), k.data_ptr(), v.data_ptr()
    a.q_strides, a.k_strides, a.v_strides = (Strides(*t.stride()[:3]) for t in (q, k, v))
    a.dtype, a.batch, a.kv_batch, a.queries, a.keys = int(dtype is torch.bfloat16), B, B, Lq, Lk
    a.heads, a.kv_heads, a.head_dim, a.scale = H, H, D, D ** -0.5
    lib = get_lib()
    assert lib.nova_cross_attention_uses_rest(a) == 1
    o, gq, gk, gv = (torch.empty_like(t) for t in (q, q, k, v))
    lse = torch.empty(B, H, Lq, device=DEV)
    n = [lib.nova_cross_attention_workspace_bytes(a, i) for i in (0, 1)]
    ws = torch.empty(max(n) + 16, dtype=torch.uint8, device=DEV)
    stream = torch.cuda.current_stream().cuda_stream
    lib.nova_cross_attention(a, o.data_ptr(), None, lse.data_ptr(), ws.data_ptr(), n[0], stream)
    lib.nova_cross_attention_backward(a, o.data_ptr(), None, lse.data_ptr(), go.data_ptr(),
                                      gq.data_ptr(), gk.data_ptr(), gv.data_ptr(), ws.data_ptr(),
                                      n[1], stream)
    assert lib.nova_get_last_error() == 0
    assert torch.equal(o, out)
    err = (gq.double() - dq).norm().item()
    assert 2 * bound < err <= _rounded_terms(q, k, v, go, u, False)[1]
