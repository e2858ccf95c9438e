"""The operators on clustered rows against their 64-bit forms (``tests/_clusters_ref.py``)."""

from __future__ import annotations

import math

import pytest
import torch

from _clusters_ref import attention_ref, order_ref, reads, select_ref

pytestmark = pytest.mark.gpu

BF, HF, F32 = torch.bfloat16, torch.float16, torch.float32


@pytest.fixture(scope="module")
def clusters(cuda_device):
    from flash_kmeans_cuda import clusters

    return clusters


@pytest.fixture(autouse=True)
def no_wait_expired():
    """No kernel of a test gave up a wait."""
    yield
    from flash_kmeans_cuda import _lib

    _lib.device_status()


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0):
    return torch.randn(*shape, generator=gen(seed), device="cuda")


def close(got, want, tol, what=""):
    got = got.double()
    fin = want.isfinite()
    assert torch.equal(got.isfinite(), fin), f"{what}: finite in other places"
    assert torch.equal(got[~fin & ~want.isnan()], want[~fin & ~want.isnan()]), what
    over = ((got - want).abs() - tol)[fin]
    assert over.numel() == 0 or over.max().item() <= 0, \
        f"{what}: {(over > 0).sum().item()} of {over.numel()} beyond the tolerance, by {over.max().item():.3g}"


# ------------------------------------------------------------------ order
@pytest.mark.parametrize("B,N,K", [(1, 1, 1), (3, 2, 5), (2, 511, 7), (1, 4096, 2046), (2, 4097, 2047), (5, 5000, 64),
                                   (1, 100003, 1), (2, 70001, 50000), (1, 300000, 511), (4, 16385, 4194305)])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_order(clusters, B, N, K, dtype):
    ids = torch.randint(-2, K + 2, (B, N), generator=gen(N + K), device="cuda").to(dtype)
    ids[:, : N // 3] = ids[:, :1]  # one long cluster
    order, offsets = clusters.cluster_order(ids, K)
    want_order, want_off = order_ref(ids, K)
    assert order.dtype == offsets.dtype == torch.int32
    assert torch.equal(order.cpu(), want_order) and torch.equal(offsets.cpu(), want_off)


def test_order_wide_ids_and_views(clusters):
    ids = torch.tensor([[0, 1 << 32, -(1 << 40), 2, 1, (1 << 32) + 2, 1 << 62]], device="cuda")
    order, offsets = clusters.cluster_order(ids, 3)
    assert order.tolist() == [[0, 4, 3, -1, -1, -1, -1]] and offsets.tolist() == [[0, 1, 2, 3]]
    wide = torch.randint(0, 9, (40, 6), device="cuda", dtype=torch.int32)
    order, offsets = clusters.cluster_order(wide.t(), 9)  # not contiguous
    want = order_ref(wide.t(), 9)
    assert torch.equal(order.cpu(), want[0]) and torch.equal(offsets.cpu(), want[1])
    order, offsets = clusters.cluster_order(torch.zeros(2, 0, dtype=torch.int32, device="cuda"), 3)
    assert order.shape == (2, 0) and offsets.tolist() == [[0] * 4] * 2
    with pytest.raises(RuntimeError, match="int32 or int64"):
        clusters.cluster_order(wide.float(), 3)
    with pytest.raises(RuntimeError, match="n_clusters"):
        clusters.cluster_order(wide, 0)


# ------------------------------------------------------------------ lookup
def lookup_check(clusters, table, ids, scale, dy):
    table = table.detach().requires_grad_(True)
    y = clusters.cluster_lookup(table, ids, scale=scale)
    (grad,) = torch.autograd.grad(y, table, dy)
    K, D = table.shape[-2:]
    three = table.detach().double().reshape(-1, K, D)
    two = ids.reshape(three.shape[0], -1).long()
    ok = (two >= 0) & (two < K)
    at = torch.where(ok, two, 0)
    sc = torch.tensor(scale, dtype=torch.float32).double().item()
    want = three.gather(1, at[..., None].expand(-1, -1, D)) * ok[..., None] * sc
    u = torch.finfo(table.dtype).eps / 2
    f = 2.0 ** -24
    tiny = {HF: 2.0 ** -24, BF: 2.0 ** -126, F32: 2.0 ** -126}[table.dtype]
    want = want.reshape(y.shape)
    assert y.dtype == grad.dtype == table.dtype
    close(y, want, (u + f) * want.abs() * (1 + u) + tiny, "y")
    d = dy.double().reshape(*two.shape, D) * ok[..., None]
    index = at[..., None].expand(-1, -1, D)
    g = torch.zeros_like(three).scatter_add_(1, index, d) * sc
    mag = torch.zeros_like(three).scatter_add_(1, index, d.abs()) * abs(sc)
    most = int(torch.zeros_like(three[..., 0]).scatter_add_(1, at, ok.double()).max().item()) if two.numel() else 0
    close(grad.reshape(g.shape), g, ((most + 2) * f * mag + u * g.abs()) * (1 + u) + tiny, "table gradient")
    again = torch.autograd.grad(clusters.cluster_lookup(table, ids, scale=scale), table, dy)[0]
    assert torch.equal(grad, again), "two runs differ"
    return y, grad


@pytest.mark.parametrize("dtype", [BF, HF, F32])
@pytest.mark.parametrize("rows,N,K,D,scale", [(0, 1, 1, 1, 1.0), (0, 333, 17, 128, 1.0), (0, 1000, 3000, 7, 0.3),
                                              (0, 5000, 40, 1024, 32.0), (0, 700, 50, 2056, -1.5), (3, 129, 5, 100, 1.0),
                                              (4, 3000, 300, 64, 2.0), (2, 20000, 3, 16, 1.0)])
def test_lookup(clusters, dtype, rows, N, K, D, scale):
    shape = (K, D) if rows == 0 else (rows, K, D)
    table = randn(*shape, seed=N).to(dtype)
    ids = torch.randint(-1, K + 1, (N,) if rows == 0 else (rows, N), generator=gen(D), device="cuda")
    ids[..., N // 2:] = K // 2  # one id holds half of the positions
    if N % 2:
        ids = ids.int()
    lookup_check(clusters, table, ids, scale, randn(*ids.shape, D, seed=5).to(dtype))


def test_lookup_views_and_empties(clusters):
    base = randn(20 * 24 + 1).to(BF)
    table = base[1:].view(20, 24)  # rows not on 16 bytes
    ids = torch.randint(0, 20, (6, 50), generator=gen(1), device="cuda").t()
    lookup_check(clusters, table, ids, 1.0, randn(50, 6, 24, seed=2).to(BF))
    lookup_check(clusters, randn(24, 20).to(HF).t(), ids, 1.0, randn(1, 6, 24, seed=2).to(HF).expand(50, 6, 24))
    t = randn(4, 8).requires_grad_(True)
    y = clusters.cluster_lookup(t, torch.zeros(0, dtype=torch.long, device="cuda"))
    assert y.shape == (0, 8) and torch.equal(torch.autograd.grad(y.sum(), t)[0], torch.zeros_like(t))
    y = clusters.cluster_lookup(t, torch.tensor(2, device="cuda"))  # one id, no dimension
    assert y.shape == (8,) and torch.equal(y, t[2])
    # out of range everywhere; infinities in rows that nothing reads
    t = torch.full((3, 8), math.inf, device="cuda", requires_grad=True)
    y = clusters.cluster_lookup(t, torch.tensor([-1, 3], device="cuda"))
    assert torch.equal(y, torch.zeros_like(y)) and torch.autograd.grad(y.sum(), t)[0].eq(0).all()
    with pytest.raises(RuntimeError, match="once"):
        t = randn(3, 8).requires_grad_(True)
        torch.autograd.grad(clusters.cluster_lookup(t, torch.tensor([1], device="cuda")).square().sum(), t, create_graph=True)


def test_lookup_gradient_against_differences(clusters):
    """The lookup is linear: <f(t + d) - f(t), w> = <grad, d>, up to fp32 rounding."""
    t, d = randn(9, 32, seed=1).requires_grad_(True), randn(9, 32, seed=2)
    ids = torch.randint(0, 9, (200,), generator=gen(3), device="cuda")
    w = randn(200, 32, seed=4)
    y = clusters.cluster_lookup(t, ids, scale=0.5)
    (g,) = torch.autograd.grad(y, t, w)
    diff = ((clusters.cluster_lookup((t + d).detach(), ids, scale=0.5).double() - y.double()) * w.double()).sum()
    # each of the 200 * 32 terms rounds t + d, the scaling and the difference: 3 * 2**-24 of their magnitudes
    bound = 4 * 2.0 ** -24 * ((t.abs() + d.abs())[ids].double() * w.abs().double()).sum() + 210 * 2.0 ** -24 * (g * d).double().abs().sum()
    assert (diff - (g.double() * d.double()).sum()).abs() <= bound


# ------------------------------------------------------------------ select
def key_clusters(R, N, K, seed, drop=0.0):
    ids = torch.randint(0, K, (R, N), generator=gen(seed), device="cuda", dtype=torch.int32)
    if drop:
        ids[torch.rand(R, N, generator=gen(seed + 1), device="cuda") < drop] = -1
    order, offsets = order_ref(ids, K)
    return ids, order.cuda(), offsets.cuda()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("B,Hkv,G,Nq,N,K,D,top", [(1, 1, 1, 1, 1, 1, 8, 1), (2, 2, 3, 5, 100, 13, 80, 5), (1, 2, 4, 70, 999, 129, 128, 16),
                                                  (3, 1, 16, 1, 4000, 1000, 64, 64), (1, 1, 5, 33, 3000, 1500, 24, 40),
                                                  (1, 2, 2, 17, 20000, 9001, 128, 1024), (1, 1, 1, 9, 50, 40, 16, 40), (1, 1, 2, 3, 50, 7, 16, 20)])
@pytest.mark.parametrize("masked", [False, True])
def test_select(clusters, dtype, B, Hkv, G, Nq, N, K, D, top, masked):
    R = B * Hkv
    q, cen = randn(B, Hkv * G, Nq, D, seed=1).to(dtype), randn(R, K, D, seed=2).to(dtype)
    _, order, offsets = key_clusters(R, N, K, 3)
    kw = {}
    if masked:
        kw["order"], kw["q_pos"] = order, torch.randint(-1, N, (B, Nq), generator=gen(4), device="cuda", dtype=torch.int32)
        kw["bias"] = (offsets[:, 1:] - offsets[:, :-1]).float().log()  # -inf where empty
        cen[offsets[:, 1:] == offsets[:, :-1]] = math.nan  # what an empty cluster holds is of no account
    got = clusters.cluster_select(q, cen, offsets, top, **kw)
    assert got.dtype == torch.int32 and torch.equal(got, select_ref(q, cen, offsets, top, **kw))


@pytest.mark.parametrize("K", [60, 700, 3000])
def test_select_ties_and_borders(clusters, K):
    """Scores that are equal, or differ by less than fp32 sums can tell."""
    D, Nq = 128, 40
    q = randn(1, 2, Nq, D, seed=1).to(HF)
    base = randn(1, 4, D, seed=2).to(HF)
    cen = base.repeat(1, K // 4, 1).contiguous()
    _, _, offsets = key_clusters(1, 50 * K, K, 3)
    got = clusters.cluster_select(q, cen, offsets, K // 3)  # runs of equal centroids cut by top_k
    assert torch.equal(got, select_ref(q, cen, offsets, K // 3))
    # one product of 2**-9 more or less beside terms near 1e4: below fp32's resolution
    big = torch.zeros(1, K, D, device="cuda", dtype=HF)
    big[..., 0] = 256.0
    big[..., 1] = torch.randint(0, 64, (1, K), generator=gen(4), device="cuda").to(HF) * 2.0 ** -14
    qq = torch.ones(1, 1, 3, D, device="cuda", dtype=HF)
    qq[..., 0] = 16384.0
    got = clusters.cluster_select(qq, big, offsets, 17)
    assert torch.equal(got, select_ref(qq, big, offsets, 17))


@pytest.mark.parametrize("K,Nq", [(90, 5), (90, 700), (700, 700), (3000, 5)])
@pytest.mark.parametrize("small", ["neither", "queries", "centroids"])
def test_select_squares_that_underflow(clusters, K, Nq, small):
    """Queries or centroids whose squares are below fp32's range: a pair of products of 2**-16 cancels and
    takes the product of 2**-48 that decides with it, and what fp32 keeps is in another order."""
    q, cen = torch.zeros(1, 1, Nq, 32, device="cuda"), torch.zeros(1, K, 32, device="cuda")
    first, second = (torch.randperm(K, generator=gen(i), device="cuda") % 64 + 1 for i in (1, 2))
    a, b = {"neither": (2.0 ** -8, 2.0 ** -8), "queries": (2.0 ** -78, 2.0 ** 62), "centroids": (2.0 ** 62, 2.0 ** -78)}[small]
    q[..., :2], cen[..., 0], cen[..., 1] = a, b, -b
    q[..., 2] = q[..., 20] = a if small == "queries" else a * 2.0 ** -32
    b = b * 2.0 ** -32 if small == "queries" else b
    cen[..., 2], cen[..., 20] = first * b, second * b * 2.0 ** -8
    q, cen = q.to(BF), cen.to(BF)
    _, _, offsets = key_clusters(1, 50 * K, K, 3)
    got = clusters.cluster_select(q, cen, offsets, K // 4)
    assert torch.equal(got, select_ref(q, cen, offsets, K // 4))


def test_select_many_queries(clusters):
    """More queries than warps at once, with ties, near ties and masks among them."""
    q = (randn(1, 4, 7001, 32, seed=1) * 2).round().div(2).to(BF)
    cen = (randn(4, 90, 32, seed=2) * 2).round().div(2).to(BF)
    cen[:, 40:50] = cen[:, 10:20]
    cen[:, 50:60] = cen[:, 20:30] + 2.0 ** -9 * randn(4, 10, 32, seed=3).sign().to(BF)
    _, order, offsets = key_clusters(4, 2000, 90, 4)
    pos = torch.randint(-1, 2000, (1, 7001), generator=gen(5), device="cuda", dtype=torch.int32)
    got = clusters.cluster_select(q, cen, offsets, 13, order=order, q_pos=pos)
    assert torch.equal(got, select_ref(q, cen, offsets, 13, order, pos))


@pytest.mark.parametrize("B,Hkv,G,Nq,K,top", [(1, 2, 1, 3001, 6001, 9), (10, 4, 1, 999, 1001, 5), (2, 1, 2, 8000, 2200, 3)])
def test_select_rounds(clusters, B, Hkv, G, Nq, K, top):
    """More scores than one round takes: rounds of a row's queries, and of rows."""
    D, R = 8, B * Hkv
    q, cen = randn(B, Hkv * G, Nq, D, seed=1).to(BF), randn(R, K, D, seed=2).to(BF)
    _, order, offsets = key_clusters(R, 5 * K, K, 3)
    pos = torch.randint(-1, 5 * K, (B, Nq), generator=gen(4), device="cuda", dtype=torch.int32)
    bias = randn(R, K, seed=5)
    got = clusters.cluster_select(q, cen, offsets, top, order=order, q_pos=pos, bias=bias)
    for r in range(R):
        b, h = divmod(r, Hkv)
        for part in torch.arange(Nq, device="cuda").split(1000):
            want = select_ref(q[b:b + 1, h * G:h * G + G, part], cen[r:r + 1], offsets[r:r + 1], top, order[r:r + 1], pos[b:b + 1, part], bias[r:r + 1])
            assert torch.equal(got[r:r + 1, part], want)


def test_select_infinities(clusters):
    q, cen = randn(1, 2, 4, 16, seed=1).to(BF), randn(1, 6, 16, seed=2).to(BF)
    offsets = torch.arange(7, device="cuda", dtype=torch.int32)[None]
    bias = torch.tensor([[0, math.inf, 0, -math.inf, math.inf, math.nan]], device="cuda")
    for top in (1, 2, 3, 6):
        got = clusters.cluster_select(q, cen, offsets, top, bias=bias)
        assert torch.equal(got, select_ref(q, cen, offsets, top, bias=bias))
    cen[0, 2, 3] = math.inf
    cen[0, 0, 0] = math.nan
    for top in (1, 2, 6):
        got = clusters.cluster_select(q, cen, offsets, top)
        assert torch.equal(got, select_ref(q, cen, offsets, top))
    q[0, 0, 1] = math.nan
    got = clusters.cluster_select(q, cen, offsets, 3)
    assert got[0, 1].tolist() == [-1, -1, -1]
    huge = torch.full((1, 1, 1, 16), 3e38, device="cuda").to(BF)  # sums past fp32
    c2 = torch.tensor([1.0, 2.0, -1.0, 3.0], device="cuda").to(BF)[None, :, None].expand(1, 4, 16).contiguous() * 2
    got = clusters.cluster_select(huge, c2, offsets[:, :5], 2)
    assert got.tolist() == [[[1, 3]]]


def test_select_refusals(clusters):
    q, cen = randn(2, 4, 3, 16).to(BF), randn(4, 6, 16).to(BF)
    offsets = torch.arange(7, device="cuda", dtype=torch.int32).repeat(4, 1)
    pos = torch.zeros(2, 3, device="cuda", dtype=torch.int32)
    call = clusters.cluster_select
    for bad, match in [((q.float(), cen, offsets, 2), "float16 or bfloat16"), ((q, cen.half(), offsets, 2), "dtype"),
                       ((q, cen[:3], offsets[:3], 2), "kv_heads"), ((q, cen, offsets[:, :5], 2), "offsets"),
                       ((q, cen, offsets.long(), 2), "int32"), ((q[..., :12], cen[..., :12], offsets, 2), "head_dim"),
                       ((q, cen, offsets, 2000), "top_k"), ((q, cen, offsets, -1), "top_k")]:
        with pytest.raises(RuntimeError, match=match):
            call(*bad)
    with pytest.raises(RuntimeError, match="order"):
        call(q, cen, offsets, 2, q_pos=pos)
    with pytest.raises(RuntimeError, match="q_pos"):
        call(q, cen, offsets, 2, order=offsets, q_pos=pos[:1])
    with pytest.raises(ValueError, match="CUDA"):
        call(q, cen, offsets.cpu(), 2)
    assert call(q, cen, offsets, 0).shape == (4, 3, 0)
    assert call(q[:, :, :0], cen, offsets, 2).shape == (4, 0, 2)


# ------------------------------------------------------------------ attention
def attention_case(B, Hkv, G, Nq, N, K, D, top, dtype, seed=0, causal=True, drop=0.1):
    R = B * Hkv
    q, k, v = (randn(B, h, n, D, seed=seed + i).to(dtype) for i, (h, n) in enumerate([(Hkv * G, Nq), (Hkv, N), (Hkv, N)]))
    _, order, offsets = key_clusters(R, N, K, seed + 3, drop)
    sel = torch.rand(R, Nq, K, generator=gen(seed + 4), device="cuda").argsort(-1)[..., :top].int()
    sel = torch.nn.functional.pad(sel, (0, top - sel.shape[-1]), value=-1).contiguous()
    sel[torch.rand(sel.shape, generator=gen(seed + 5), device="cuda") < 0.1] = -1
    pos = (torch.arange(Nq, device="cuda", dtype=torch.int32) + (N - Nq)).repeat(B, 1) if causal else None
    if causal and Nq > 3:
        pos[:, 1] = -1  # sees nothing
    return q, k, v, sel, order, offsets, pos


def attention_check(clusters, q, k, v, sel, order, offsets, pos, scale=None, seed=9):
    q, k, v = (t.detach().requires_grad_(True) for t in (q, k, v))
    out, lse = clusters.cluster_attention(q, k, v, sel, order, offsets, q_pos=pos, scale=scale, return_lse=True)
    dout = randn(*q.shape, seed=seed).to(q.dtype)
    grads = torch.autograd.grad(out, (q, k, v), dout)
    val, tol = attention_ref(q.detach(), k.detach(), v.detach(), sel, order, offsets, pos, scale, dout)
    close(out.detach(), val["out"], tol["out"], "out")
    close(lse, val["lse"], tol["lse"], "lse")
    for name, g, like in zip(("dq", "dk", "dv"), grads, (q, k, v)):
        assert g.dtype == like.dtype and g.shape == like.shape
        close(g, val[name], tol[name], name)
    with torch.no_grad():
        assert torch.equal(out, clusters.cluster_attention(q, k, v, sel, order, offsets, q_pos=pos, scale=scale))
    out2 = clusters.cluster_attention(q, k, v, sel, order, offsets, q_pos=pos, scale=scale)
    for g, h in zip(grads, torch.autograd.grad(out2, (q, k, v), dout)):
        assert torch.equal(g, h), "two runs differ"
    return out, grads


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("B,Hkv,G,Nq,N,K,D,top", [
    (1, 1, 1, 1, 1, 1, 8, 1), (1, 1, 1, 2, 17, 1, 64, 1), (2, 2, 3, 37, 100, 7, 80, 3), (1, 2, 4, 130, 130, 5, 128, 2),
    (1, 1, 8, 20, 500, 9, 128, 9), (2, 1, 16, 9, 300, 20, 64, 6), (1, 1, 20, 5, 200, 6, 72, 4), (1, 2, 9, 33, 129, 11, 128, 7),
    (1, 1, 2, 1, 5000, 40, 128, 30), (3, 2, 4, 1, 2000, 31, 64, 40), (1, 1, 1, 300, 64, 64, 16, 10)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention(clusters, dtype, B, Hkv, G, Nq, N, K, D, top, causal):
    if causal and Nq > N:
        pytest.skip("positions before the first key")
    attention_check(clusters, *attention_case(B, Hkv, G, Nq, N, K, D, top, dtype, seed=Nq + D, causal=causal))


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("B,Hkv,G,Nq,N,K,D,top", [(1, 2, 4, 700, 1500, 23, 128, 7), (2, 1, 3, 1001, 1300, 17, 72, 5),
                                                  (1, 1, 16, 400, 2500, 30, 64, 9), (2, 2, 1, 3000, 3001, 100, 32, 5),
                                                  (1, 1, 24, 300, 1500, 9, 128, 9), (1, 2, 2, 2000, 2100, 40, 8, 6),
                                                  (1, 1, 5, 900, 1300, 20, 104, 6), (3, 1, 2, 1700, 1700, 6, 64, 3)])
@pytest.mark.parametrize("causal", [False, True])
def test_attention_many_queries(clusters, dtype, B, Hkv, G, Nq, N, K, D, top, causal):
    attention_check(clusters, *attention_case(B, Hkv, G, Nq, N, K, D, top, dtype, seed=Nq + D, causal=causal))


def many(seed=5, dtype=BF, **kw):
    """A case of the form by clusters: 1000 queries, two sequences."""
    return attention_case(2, 1, 4, 1000, 1500, 15, 64, 5, dtype, seed=seed, **kw)


def test_many_queries_same_cluster_twice(clusters):
    q, k, v, sel, order, offsets, pos = many(drop=0.0)
    sel[..., 2] = sel[..., 0]
    attention_check(clusters, q, k, v, sel, order, offsets, pos)


def test_many_queries_bad_entries_read_nothing(clusters):
    q, k, v, sel, order, offsets, pos = many(drop=0.0)
    sel[0, :, 0] = 15
    sel[1, :, 0] = -(1 << 31)
    sel[1, :, 1] = (1 << 31) - 1
    order[0, 5], order[1, 7], order[1, 9] = 1500, -5, (1 << 31) - 1
    attention_check(clusters, q, k, v, sel, order, offsets, pos)


def test_many_queries_empty_clusters_and_blind_queries(clusters):
    q, k, v, sel, order, offsets, pos = many()
    offsets[:, 4:] = offsets[:, 4:5]  # the clusters from the fourth on are empty
    pos[:, 100:400] = -1
    sel[:, 500:600] = -1
    attention_check(clusters, q, k, v, sel, order, offsets, pos)
    pos[:] = -1
    attention_check(clusters, q, k, v, sel, order, offsets, pos)


def test_many_queries_strided_inputs(clusters):
    q, k, v, sel, order, offsets, pos = many(drop=0.0)
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    out, _ = attention_check(clusters, *turned, sel, order, offsets, pos)
    padded = [torch.nn.functional.pad(t, (0, 8))[..., :64] for t in (q, k, v)]
    assert torch.equal(out, attention_check(clusters, *padded, sel, order, offsets, pos)[0])
    odd = [torch.nn.functional.pad(t, (0, 3))[..., :64] for t in (q, k, v)]
    assert torch.equal(out, attention_check(clusters, *odd, sel, order, offsets, pos)[0])


def test_many_queries_some_gradients_only(clusters):
    q, k, v, sel, order, offsets, pos = many()
    _, full = attention_check(clusters, q, k, v, sel, order, offsets, pos)
    dout = randn(*q.shape, seed=9).to(BF)
    for which in ((0,), (1,), (0, 2)):
        a = [t.detach().requires_grad_(i in which) for i, t in enumerate((q, k, v))]
        out = clusters.cluster_attention(*a, sel, order, offsets, q_pos=pos)
        for i, g in zip(which, torch.autograd.grad(out, [a[i] for i in which], dout)):
            assert torch.equal(g, full[i])


@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_many_queries_masked_places_hold_anything(clusters, what):
    q, k, v, sel, order, offsets, pos = many()
    pos[1, 500:] = -1
    pos.clamp_(max=1200)
    k[:, :, 1201:] = what
    v[:, :, 1201:] = what
    q[1, :, 500:] = what
    sees = (pos >= 0)[:, None, :, None]
    val, tol = attention_ref(q, k, v, sel, order, offsets, pos, None, torch.ones_like(q))
    a = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = clusters.cluster_attention(*a, sel, order, offsets, q_pos=pos)
    grads = torch.autograd.grad(out, a, torch.where(sees, 1.0, what).to(BF).expand_as(q).contiguous())
    close(out.detach(), val["out"], tol["out"], "out")
    close(grads[1], val["dk"], tol["dk"], "dk")
    close(grads[2], val["dv"], tol["dv"], "dv")
    live = sees.expand_as(q)
    close(grads[0][live], val["dq"][live], tol["dq"][live], "dq")
    assert grads[0][~live].eq(0).all()


@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("case", [(2, 1, 3, 1001, 1300, 17, 72, 5), (1, 2, 4, 700, 1500, 23, 128, 7), (1, 1, 16, 400, 2500, 30, 64, 9),
                                  (2, 1, 3, 40, 200, 7, 64, 3), (1, 2, 5, 70, 700, 3, 128, 2)])
@pytest.mark.parametrize("dtype", [BF, HF])
def test_what_some_do_not_see_holds_anything(clusters, dtype, case, what):
    """A key, a query and a gradient of out that are not finite show only where they are read."""
    q, k, v, sel, order, offsets, pos = attention_case(*case, dtype, seed=3)
    B, Hkv, N, Nq = case[0], case[1], case[4], case[3]
    dout = randn(*q.shape, seed=8).to(dtype)
    read = reads(sel, order, offsets, pos, Hkv) > 0                      # (R, Nq, N)
    odd = torch.zeros_like(read[..., 0])
    odd[:, [Nq // 3, Nq - 2]] = True                                     # odd queries
    odd |= read[:, :, [N - 30, N - Nq // 5]].any(-1)                     # and those that read odd keys
    spoilt = (read & odd[..., None]).any(1).view(B, Hkv, N)              # keys that an odd query reads
    odd = odd.view(B, Hkv, 1, Nq).expand(B, Hkv, case[2], Nq).reshape(q.shape[:3])
    assert not odd.all() and not spoilt.all()
    val, tol = attention_ref(q, k, v, sel, order, offsets, pos, None, dout.masked_fill(odd[..., None], 0.0))
    for t in (k, v):
        t[:, :, [N - 30, N - Nq // 5]] = what
    q[:, :, Nq // 3] = what
    dout[:, :, Nq - 2] = what
    a = [t.requires_grad_(True) for t in (q, k, v)]
    out, lse = clusters.cluster_attention(*a, sel, order, offsets, q_pos=pos, return_lse=True)
    dq, dk, dv = torch.autograd.grad(out, a, dout)
    for name, got, keep in (("out", out, ~odd), ("lse", lse, ~odd), ("dq", dq, ~odd), ("dk", dk, ~spoilt), ("dv", dv, ~spoilt)):
        close(got.detach()[keep], val[name][keep], tol[name][keep], name)


def test_many_queries_far_apart_values(clusters):
    """Rows of out whose magnitudes differ by 2**60 and more: parts keep a power of two each."""
    q, k, v, sel, order, offsets, pos = many(drop=0.0)
    v = (v.float() * torch.exp2(torch.randint(-60, 61, (2, 1, 1500, 1), generator=gen(8), device="cuda").float())).to(BF)
    out, lse = clusters.cluster_attention(q, k, v, sel, order, offsets, q_pos=pos, return_lse=True)
    val, tol = attention_ref(q, k, v, sel, order, offsets, pos)
    close(out, val["out"], tol["out"], "out")
    close(lse, val["lse"], tol["lse"], "lse")


def test_many_queries_two_streams_at_once(clusters):
    """Two calls that run beside each other, and a captured one replayed beside an eager one."""
    a, b = many(seed=5), many(seed=50)

    def step(c):
        leaves = [t.detach().requires_grad_(True) for t in c[:3]]
        out = clusters.cluster_attention(*leaves, *c[3:6], q_pos=c[6])
        return (out.detach(), *torch.autograd.grad(out, leaves, torch.ones_like(out)))

    want = [step(a), step(b)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(3):
        for c, s in zip((a, b), streams):
            with torch.cuda.stream(s):
                got.append(step(c))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        for x, y in zip(g, want[i % 2]):
            assert torch.equal(x, y)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = step(a)
    graph.replay()
    eager = step(b)
    torch.cuda.synchronize()
    for x, y in zip(held + eager, want[0] + want[1]):
        assert torch.equal(x, y)


def test_attention_rounds(clusters):
    """So many parts that the queries are taken in rounds."""
    q, k, v, sel, order, offsets, pos = attention_case(1, 4, 32, 300, 17500, 128, 128, 128, BF)
    out, lse = clusters.cluster_attention(q, k, v, sel, order, offsets, q_pos=pos, return_lse=True)
    for h in range(4):
        heads, row = slice(32 * h, 32 * h + 32), slice(h, h + 1)
        val, tol = attention_ref(q[:, heads], k[:, row], v[:, row], sel[row], order[row], offsets[row], pos)
        close(out[:, heads], val["out"], tol["out"], "out")
        close(lse[:, heads], val["lse"], tol["lse"], "lse")


def test_positions_of_any_size(clusters):
    """q_pos far behind the last key, and below zero."""
    for args in (attention_case(1, 1, 2, 40, 100, 6, 64, 4, BF), attention_case(1, 1, 4, 900, 900, 12, 64, 6, BF)):
        q, k, v, sel, order, offsets, pos = args
        pos[:, ::3] = (1 << 31) - 1
        pos[:, 1::3] = -(1 << 31)
        attention_check(clusters, q, k, v, sel, order, offsets, pos)
        K = offsets.shape[1] - 1
        cen = randn(1, K, 64, seed=8).to(BF)
        offsets[:, 3:] = offsets[:, 3:4]  # empty clusters behind the third
        got = clusters.cluster_select(q, cen, offsets, 5, order=order, q_pos=pos)
        assert torch.equal(got, select_ref(q, cen, offsets, 5, order, pos))


def test_attention_large_clusters(clusters):
    """Clusters of many key tiles, one of them selected by every query."""
    q, k, v, sel, order, offsets, pos = attention_case(1, 1, 4, 400, 3000, 4, 64, 2, BF, drop=0.0)
    sel[..., 0] = 2
    sel[..., 1] = torch.where(sel[..., 1] == 2, 3, sel[..., 1])
    attention_check(clusters, q, k, v, sel, order, offsets, pos)


@pytest.mark.parametrize("top", [1, 2])
@pytest.mark.parametrize("Nq", [2, 400])
def test_query_gradient_of_close_keys(clusters, Nq, top):
    """Keys of a cluster that lie close together: the gradient of q keeps the accuracy of its last
    rounding, at most 2**-8 of its norm (the scores' errors, some 2**-13, and dS's 2**-17 stay below 2**-10)."""
    q, k, v, _, order, offsets, _ = attention_case(1, 2, 4, Nq, 500, 16, 128, top, BF, causal=False, drop=0.0)
    for r in range(2):
        for c in range(16):
            rows = order[r, offsets[r, c]:offsets[r, c + 1]].long()
            k[0, r, rows] = (randn(1, 128, seed=100 + c) + 0.5 * k[0, r, rows].float()).to(BF)
    sel = torch.randint(0, 16 - top, (2, Nq, 1), generator=gen(1), device="cuda", dtype=torch.int32) + torch.arange(top, device="cuda", dtype=torch.int32)
    dout = randn(*q.shape, seed=9).to(BF)
    val, _ = attention_ref(q, k, v, sel, order, offsets, None, None, dout)
    q.requires_grad_(True)
    (dq,) = torch.autograd.grad(clusters.cluster_attention(q, k, v, sel, order, offsets), q, dout)
    off = ((dq.double() - val["dq"]).norm() / val["dq"].norm()).item()
    assert off <= 2.0 ** -8 + 2.0 ** -10, off


def test_attention_scores_far_apart(clusters):
    """Weights that span the whole range; a scale of its own, a negative one too."""
    for scale in (3.0, -0.5):
        attention_check(clusters, *attention_case(1, 1, 4, 50, 200, 8, 64, 4, BF, seed=3), scale=scale)


def test_attention_same_cluster_twice(clusters):
    q, k, v, sel, order, offsets, pos = attention_case(1, 2, 2, 40, 100, 6, 64, 4, HF, drop=0.0)
    sel[..., 2] = sel[..., 0]
    attention_check(clusters, q, k, v, sel, order, offsets, pos)


def test_attention_strided_inputs(clusters):
    """(batch, positions, heads, head_dim) views; rows that are not on 16 bytes; broadcast keys."""
    q, k, v, sel, order, offsets, pos = attention_case(2, 2, 2, 30, 90, 5, 64, 3, BF, drop=0.0)
    turned = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k, v)]
    attention_check(clusters, *turned, sel, order, offsets, pos)
    odd = [torch.nn.functional.pad(t, (0, 3))[..., :64] for t in (q, k, v)]
    attention_check(clusters, *odd, sel, order, offsets, pos)
    off = torch.empty(q.numel() + 1, device="cuda", dtype=BF)[1:].view(q.shape).copy_(q)
    attention_check(clusters, off, k, v, sel, order, offsets, pos)
    one = k[:, :1].detach().requires_grad_(True)
    out = clusters.cluster_attention(q, one.expand(2, 2, 90, 64), v, sel, order, offsets, q_pos=pos)
    dout = randn(*q.shape, seed=9).to(BF)
    (g,) = torch.autograd.grad(out, one, dout)
    val, tol = attention_ref(q, k[:, :1].expand(2, 2, 90, 64), v, sel, order, offsets, pos, None, dout)
    want, room = val["dk"].sum(1, keepdim=True), tol["dk"].sum(1, keepdim=True)
    close(g, want, room + 2.0 ** -8 * want.abs(), "broadcast key gradient")


@pytest.mark.parametrize("what", [math.nan, math.inf])
def test_attention_masked_places_hold_anything(clusters, what):
    """NaN or infinities in keys that no query sees and in queries that see nothing."""
    q, k, v, sel, order, offsets, pos = attention_case(2, 1, 3, 40, 200, 7, 64, 3, BF)
    pos[1, 10:] = -1
    pos[:, :10] = pos[:, :10].clamp(max=150)
    pos.clamp_(max=150)
    k[:, :, 151:] = what
    v[:, :, 151:] = what
    q[1, :, 10:] = what
    sees = (pos >= 0)[:, None, :, None]
    val, tol = attention_ref(q, k, v, sel, order, offsets, pos, None, torch.ones_like(q))
    a = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = clusters.cluster_attention(*a, sel, order, offsets, q_pos=pos)
    dout = torch.where(sees, 1.0, what).to(BF).expand_as(q).contiguous()
    grads = torch.autograd.grad(out, a, dout)
    close(out.detach(), val["out"], tol["out"], "out")
    close(grads[1], val["dk"], tol["dk"], "dk")
    close(grads[2], val["dv"], tol["dv"], "dv")
    live = sees.expand_as(q)
    close(grads[0][live], val["dq"][live], tol["dq"][live], "dq")
    assert grads[0][~live].eq(0).all()


def test_attention_bad_entries_read_nothing(clusters):
    """Cluster ids and positions outside their ranges select nothing."""
    q, k, v, sel, order, offsets, pos = attention_case(1, 2, 2, 20, 100, 6, 64, 4, BF, drop=0.0)
    sel[0, :, 0] = 6
    sel[1, :, 0] = -(1 << 31)
    sel[1, :, 1] = (1 << 31) - 1
    order[0, 5], order[1, 7], order[1, 9] = 100, -5, (1 << 31) - 1
    attention_check(clusters, q, k, v, sel, order, offsets, pos)


def test_attention_nothing(clusters):
    q, k, v, sel, order, offsets, pos = attention_case(1, 1, 2, 4, 10, 3, 16, 2, BF)
    none = [(q, k, v, sel[..., :0], order, offsets), (q, k[:, :, :0], v[:, :, :0], sel, order[:, :0], offsets * 0),
            (q, k, v, torch.full_like(sel, -1), order, offsets)]
    for args in none:
        a = [t.detach().requires_grad_(True) for t in args[:3]]
        out, lse = clusters.cluster_attention(*a, *args[3:], return_lse=True)
        assert out.eq(0).all() and lse.eq(-math.inf).all()
        for g, t in zip(torch.autograd.grad(out, a, torch.ones_like(out)), a):
            assert g.shape == t.shape and g.eq(0).all()
    assert clusters.cluster_attention(q[:, :, :0], k, v, sel[:, :0], order, offsets).shape == (1, 2, 0, 16)


def test_attention_some_gradients_only(clusters):
    q, k, v, sel, order, offsets, pos = attention_case(1, 2, 2, 20, 100, 6, 64, 4, BF)
    _, full = attention_check(clusters, q, k, v, sel, order, offsets, pos)
    dout = randn(*q.shape, seed=9).to(BF)
    for which in ((0,), (1,), (2,), (1, 2), (0, 2)):
        a = [t.detach().requires_grad_(i in which) for i, t in enumerate((q, k, v))]
        out = clusters.cluster_attention(*a, sel, order, offsets, q_pos=pos)
        got = torch.autograd.grad(out, [a[i] for i in which], dout)
        for i, g in zip(which, got):
            assert torch.equal(g, full[i])
    with pytest.raises(RuntimeError, match="once"):
        out = clusters.cluster_attention(q.requires_grad_(True), k, v, sel, order, offsets)
        torch.autograd.grad(out.float().square().sum(), q, create_graph=True)


def test_attention_gradient_against_differences(clusters):
    """Central differences of a smooth case: dq along one direction. The step's own errors:
    out is rounded to fp16 (2**-11) on both sides of a step of 2**-4."""
    q, k, v, sel, order, offsets, _ = attention_case(1, 1, 1, 6, 60, 3, 32, 2, HF, drop=0.0)
    w, d = randn(*q.shape, seed=20).to(HF), (randn(*q.shape, seed=21).sign() * 2.0 ** -4).to(HF)
    a = q.detach().requires_grad_(True)
    out = clusters.cluster_attention(a, k, v, sel, order, offsets)
    (g,) = torch.autograd.grad(out, a, w)

    def f(x):
        return (clusters.cluster_attention(x, k, v, sel, order, offsets).double() * w.double()).sum((1, 2, 3))

    up, down = (q.double() + d.double()).half(), (q.double() - d.double()).half()
    diff = (f(up) - f(down)).item()
    along = (g.double() * (up.double() - down.double())).sum().item()
    val, tol = attention_ref(q, k, v, sel, order, offsets, None, None, w)
    # third-order term: |s| moves by at most h per key, h = scale * |d| * |k|
    h = 32 ** -0.5 * d.double().norm(dim=-1).max() * k.double().norm(dim=-1).max()
    spread = (v.double().abs().amax() * w.double().abs().sum()).item()
    bound = 2 * (tol["out"] * w.double().abs()).sum().item() + 2 * (tol["dq"] * d.double().abs()).sum().item() + 2 * h.item() ** 3 * spread
    assert abs(diff - along) <= bound


def test_attention_refusals(clusters):
    q, k, v, sel, order, offsets, pos = attention_case(2, 2, 2, 6, 30, 3, 16, 2, BF)
    call = clusters.cluster_attention
    for bad, match in [((q.float(), k.float(), v.float(), sel, order, offsets), "float16 or bfloat16"),
                       ((q, k.half(), v, sel, order, offsets), "dtype"), ((q, k, v[:, :, :9], sel, order, offsets), "same sizes"),
                       ((q[:, :3], k, v, sel, order, offsets), "kv_heads"), ((q, k, v, sel[:3], order, offsets), "sel"),
                       ((q, k, v, sel.long(), order, offsets), "int32"), ((q, k, v, sel, order[:, :9], offsets), "order"),
                       ((q, k, v, sel, order, offsets[:2]), "offsets"), ((q[0], k, v, sel, order, offsets), "q must be"),
                       ((q, k[..., :8], v, sel, order, offsets), "k must be")]:
        with pytest.raises(RuntimeError, match=match):
            call(*bad)
    with pytest.raises(RuntimeError, match="q_pos"):
        call(q, k, v, sel, order, offsets, q_pos=pos[:, :3])
    with pytest.raises(ValueError, match="CUDA"):
        call(q, k, v, sel.cpu(), order, offsets)


# ------------------------------------------------------------------ together, streams, graphs
def test_cluster_select_attend_and_train(clusters):
    """The path of a model: cluster the keys, order them, select, attend; and read centroids back."""
    from flash_kmeans_cuda import batch_kmeans_Euclid

    B, Hkv, G, N, D, K, top = 2, 2, 4, 600, 64, 12, 4
    q, v = randn(B, Hkv * G, 50, D, seed=1).to(BF), randn(B, Hkv, N, D, seed=2).to(BF)
    k = (randn(B, Hkv, 1, D, seed=3) + randn(B, Hkv, N, D, seed=4)).to(BF)
    ids, centroids, _ = batch_kmeans_Euclid(k.reshape(B * Hkv, N, D), K, max_iters=5)
    order, offsets = clusters.cluster_order(ids, K)
    pos = torch.arange(N - 50, N, device="cuda", dtype=torch.int32).repeat(B, 1)
    sel = clusters.cluster_select(q, centroids, offsets, top, order=order, q_pos=pos)
    assert torch.equal(sel, select_ref(q, centroids, offsets, top, order, pos))
    attention_check(clusters, q, k, v, sel, order, offsets, pos)
    # with every cluster selected it is causal attention over all keys
    every = torch.arange(K, device="cuda", dtype=torch.int32).expand(B * Hkv, 50, K).contiguous()
    out = clusters.cluster_attention(q, k, v, every, order, offsets, q_pos=pos).double()
    s = q.double() @ k.double().repeat_interleave(G, 1).transpose(-1, -2) * D ** -0.5
    s = s.masked_fill(torch.arange(N, device="cuda")[None, None, None] > pos[:, None, :, None], -math.inf)
    want = s.softmax(-1) @ v.double().repeat_interleave(G, 1)
    # weights and out rounded: 2**-8 of the sums of magnitudes each, the rest far below
    room = 3 * 2.0 ** -8 * (s.softmax(-1) @ v.double().abs().repeat_interleave(G, 1))
    assert ((out - want).abs() <= room).all()
    lookup_check(clusters, centroids, ids, 1.0, randn(B * Hkv, N, D, seed=6).to(BF))


def test_other_stream_and_graph_replay(clusters):
    """The calls follow the current stream; a captured step replays on new inputs, eager results beside it."""
    q, k, v, sel, order, offsets, pos = attention_case(1, 2, 4, 64, 300, 8, 64, 3, BF)
    table, ids = randn(40, 64, seed=1).to(BF), torch.randint(0, 40, (500,), device="cuda", dtype=torch.int32)
    dy, dout = randn(500, 64, seed=2).to(BF), randn(*q.shape, seed=3).to(BF)
    cen = randn(2, 8, 64, seed=7).to(BF)

    def step(q, k, v, table):
        a = [t.detach().requires_grad_(True) for t in (q, k, v, table)]
        o, f = clusters.cluster_order(ids[None], 40)
        picked = clusters.cluster_select(a[0].detach(), cen, offsets, 3, order=order, q_pos=pos)
        out = clusters.cluster_attention(*a[:3], picked, order, offsets, q_pos=pos)
        y = clusters.cluster_lookup(a[3], ids)
        return (o, f, picked, out.detach(), y.detach(), *torch.autograd.grad([out, y], a, [dout, dy]))

    eager = step(q, k, v, table)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(q, k, v, table)
    torch.cuda.current_stream().wait_stream(side)
    for x, y in zip(eager, other):
        assert torch.equal(x, y)
    held = [t.clone() for t in (q, k, v, table)]
    graphs = []
    for _ in range(2):  # two captures, each with its own scratch
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got = step(*held)
        graphs.append((g, got))
    fresh = [randn(*t.shape, seed=30 + i).to(BF) for i, t in enumerate(held)]
    for h, f in zip(held, fresh):
        h.copy_(f)
    want = step(*fresh)
    for g, _ in graphs:
        g.replay()
    torch.cuda.synchronize()
    for _, got in graphs:
        for x, y in zip(got, want):
            assert torch.equal(x, y)


def test_many_queries_offsets_of_no_grouping(clusters):
    """Offsets whose clusters overlap have more key tiles than a grouping can have: their row's keys get
    no gradient, the other rows' results stay."""
    q, k, v, sel, order, offsets, pos = attention_case(1, 3, 4, 1000, 1500, 40, 64, 5, BF, causal=False, drop=0.0)
    dout = randn(*q.shape, seed=9).to(BF)
    val, tol = attention_ref(q, k, v, sel, order, offsets, None, None, dout)
    offsets[1, 0::2], offsets[1, 1::2] = 0, 1500  # every other cluster has all keys: 240 tiles, 51 have room
    a = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = clusters.cluster_attention(*a, sel, order, offsets)
    got = dict(zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, a, dout))))
    for name, x in got.items():
        n = x.shape[1] // 3
        for rows in (slice(0, n), slice(2 * n, 3 * n)):
            close(x[:, rows], val[name][:, rows], tol[name][:, rows], name)
        assert x.isfinite().all()
    assert got["dk"][:, 1].eq(0).all() and got["dv"][:, 1].eq(0).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("causal", [False, True])
def test_many_queries_columns_stand_alone(clusters, dtype, D, causal):
    """One column holds infinities and others lie far apart: each keeps the accuracy of its own last
    rounding, 2**-8 of a bf16 column's norm at most (2**-11 fp16), P and dS rounded as much once more."""
    q, k, v, sel, order, offsets, pos = attention_case(2, 1, 4, 1000, 1500, 15, D, 5, dtype, seed=5, causal=causal, drop=0.0)
    u = torch.finfo(dtype).eps / 2
    wide = 50 if dtype == BF else 10
    power = torch.exp2(torch.randint(-wide, wide + 1, (D,), generator=gen(8), device="cuda").float())
    power[:2] = 1.0
    q[..., 2::2] = 0  # the scores come from the other half: columns of k there may be anything
    k[..., 2::2] = (k[..., 2::2].float() * power[2::2]).to(dtype)
    dout = torch.where(power == 1.0, randn(*q.shape, seed=9), torch.zeros((), device="cuda")).to(dtype)
    v = (v.float() * power).to(dtype)
    val, _ = attention_ref(q, k, v, sel, order, offsets, pos, None, dout)
    dout[..., 0] = 0
    val["dq"] = attention_ref(q, k, v, sel, order, offsets, pos, None, dout)[0]["dq"]
    holed = v.clone()
    holed[:, :, 700:1300:3, 0] = math.inf
    a = [t.detach().requires_grad_(True) for t in (q, k, v)]
    (dq,) = torch.autograd.grad(clusters.cluster_attention(*a, sel, order, offsets, q_pos=pos), a[0], dout)
    out = clusters.cluster_attention(q, k, holed, sel, order, offsets, q_pos=pos)

    def columns(got, want, what):
        off, norm = ((x.double() ** 2).sum((0, 1, 2)).sqrt() for x in (got.double() - want, want))
        step = {BF: 0.0, HF: 2.0 ** -25}[dtype] * math.sqrt(want[..., 0].numel())  # fp16's smallest values
        assert (off <= 2 * u * norm + step).all(), (what, (off / norm).tolist())

    columns(out[..., 1:], val["out"][..., 1:], "out")
    columns(dq, val["dq"], "dq")
    read = reads(sel, order, offsets, pos, 1)[:, :, 700:1300:3].any(-1)[:, None].expand(out.shape[:3])
    assert out[..., 0][read].eq(math.inf).all() and out[..., 0][~read].isfinite().all()


def test_forward_mode_tangents_are_refused(clusters):
    q, k, v, sel, order, offsets, pos = attention_case(1, 1, 2, 4, 30, 3, 16, 2, BF)
    t, ids = randn(5, 8), torch.tensor([1, 4], device="cuda")
    with torch.autograd.forward_ad.dual_level():
        dual = lambda x: torch.autograd.forward_ad.make_dual(x, torch.ones_like(x))
        for x in (t, t.detach().requires_grad_(True)):
            with pytest.raises(RuntimeError, match="tangent"):
                clusters.cluster_lookup(dual(x), ids)
        for i in range(3):
            args = [dual(x) if i == j else x for j, x in enumerate((q, k, v))]
            with pytest.raises(RuntimeError, match="tangent"):
                clusters.cluster_attention(*args, sel, order, offsets)
        assert torch.equal(clusters.cluster_lookup(t, ids), t[ids])


@pytest.mark.parametrize("offset", [0.0, 3.0, 30.0])
@pytest.mark.parametrize("Nq,top,one", [(30, 1, False), (30, 8, False), (700, 1, False), (700, 2, False), (700, 4, False), (700, 8, False), (700, 16, False),
                                        (700, 8, True)])
def test_query_gradient_of_keys_with_an_offset(clusters, Nq, top, one, offset):
    """Close keys within clusters and an offset that all keys share, as channel means of a cache: dQ keeps the
    accuracy of its last rounding (2**-8 of its norm at most). delta is summed from the same P and dP, so dS
    sums to zero but for the errors of P's sum, 2**-18 of it, and of dS's 2**-17: 2**-12 of the norm at 30 times
    the spread and 64 keys, below the 2**-10 that the scores' errors, some 2**-13 a weight, have."""
    q, k, v, _, order, offsets, _ = attention_case(1, 2, 4, Nq, 2000, 32, 128, top, BF, causal=False, drop=0.0)
    common = offset * randn(128, seed=50)
    for r in range(2):
        for c in range(32):
            rows = order[r, offsets[r, c]:offsets[r, c + 1]].long()
            k[0, r, rows] = (randn(1, 128, seed=100 + c) + 0.5 * k[0, r, rows].float() + common).to(BF)
    sel = torch.randint(0, 33 - top, (2, Nq, 1), generator=gen(1), device="cuda", dtype=torch.int32) + torch.arange(top, device="cuda", dtype=torch.int32)
    if one:
        sel[..., 1:] = -1
    dout = randn(*q.shape, seed=9).to(BF)
    val, tol = attention_ref(q, k, v, sel, order, offsets, None, None, dout)
    a = [t.requires_grad_(True) for t in (q, k, v)]
    for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(clusters.cluster_attention(*a, sel, order, offsets), a, dout)):
        off = ((g.double() - val[name]).norm() / val[name].norm()).item()
        assert off <= 2.0 ** -8 + 2.0 ** -10, (name, off)


@pytest.mark.parametrize("Nq,top", [(40, 2), (1000, 3)])
@pytest.mark.parametrize("size", [1e-3, 1e-4, 4096.0])
def test_gradients_of_fp16_far_from_one(clusters, Nq, top, size):
    """dout far from 1, some queries 2**10 times farther: P and dS leave fp16's range, the gradients do not.
    Each keeps the accuracy of two roundings, 2**-11 of the norm, beside fp16's least step in its values."""
    q, k, v, sel, order, offsets, _ = attention_case(2, 1, 4, Nq, 1500, 6, 64, top, HF, causal=False, drop=0.0)
    dout = randn(*q.shape, seed=9) * size
    if size < 1:
        k = k * 8  # and large keys, that dQ stays above fp16's least values
        q = q / 8
        dout[:, :, ::7] *= 2.0 ** -10
    else:
        q, k = q / 64, k / 64
    dout = dout.to(HF)
    val, _ = attention_ref(q, k, v, sel, order, offsets, None, None, dout)
    a = [t.detach().requires_grad_(True) for t in (q, k, v)]
    for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(clusters.cluster_attention(*a, sel, order, offsets), a, dout)):
        want = val[name]
        off, room = (g.double() - want).norm(), 2.0 ** -10 * want.norm() + 2.0 ** -25 * math.sqrt(want.numel())
        assert off <= room, (name, (off / want.norm()).item(), (room / want.norm()).item())


def test_fp16_products_past_its_range(clusters):
    """dP far above 65504, and a query whose other keys' weights are all 0."""
    for Nq in (40, 1000):
        q, k, v, sel, order, offsets, _ = attention_case(2, 1, 4, Nq, 1500, 6, 64, 3, HF, causal=False, drop=0.0)
        k[:, :, ::2] *= 2.0 ** -8
        k[:, :, 1::2] *= 2.0 ** -7
        v, dout = v * 64, (randn(*q.shape, seed=9) * 4096).to(HF)
        val, _ = attention_ref(q, k, v, sel, order, offsets, None, None, dout)
        a = q.detach().requires_grad_(True)
        (g,) = torch.autograd.grad(clusters.cluster_attention(a, k, v, sel, order, offsets), a, dout)
        assert (g.double() - val["dq"]).norm() <= 2.0 ** -10 * val["dq"].norm()
        # scores of +-2000: one key has all of the weight, and its dP is 0
        k[:] = k.sign() / 4
        k[:, :, 0] = 16.0
        q[:] = 8.0
        v[:, :, 0] = 0
        sel[..., 0] = torch.searchsorted(offsets[:, 1:].contiguous(), (order == 0).int().argmax(1, keepdim=True).int(), right=True)[:, :, None].int()[..., 0]
        val, tol = attention_ref(q, k, v, sel, order, offsets, None, None, dout)
        a = [t.detach().requires_grad_(True) for t in (q, k, v)]
        out = clusters.cluster_attention(*a, sel, order, offsets)
        for name, g in zip(("dq", "dk", "dv"), torch.autograd.grad(out, a, dout)):
            held = val[name].abs() + tol[name] <= 65504  # what fp16 can hold: dv of the one key is larger in places
            close(g[held], val[name][held], tol[name][held], name)
            assert not g.isnan().any()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("case", [(1, 2, 4, 30, 700, 9, 128, 3), (2, 1, 3, 900, 1300, 17, 80, 5), (1, 1, 16, 400, 2500, 30, 64, 9)])
def test_attention_is_off_by_its_last_rounding(clusters, dtype, case):
    """What comes before it (two terms of P and dS, 2**-16; parts, 2**-16; fp32 sums and scores) stays below
    a fifth of the last rounding, whose error is 2**-9.2 of the norm with bf16 and 2**-12.2 with fp16: together
    no more than sqrt(1 + 0.04) of it."""
    q, k, v, sel, order, offsets, pos = attention_case(*case, dtype, seed=2)
    dout = randn(*q.shape, seed=9).to(dtype)
    val, _ = attention_ref(q, k, v, sel, order, offsets, pos, None, dout)
    a = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = clusters.cluster_attention(*a, sel, order, offsets, q_pos=pos)
    for name, got in zip(("out", "dq", "dk", "dv"), (out.detach(), *torch.autograd.grad(out, a, dout))):
        off, least = (got.double() - val[name]).norm(), (val[name].to(dtype).double() - val[name]).norm()
        assert off <= 1.02 * least, (name, (off / least).item())


def test_lookup_of_no_row_is_zero_whatever_the_scale(clusters):
    t, ids = randn(5, 24).to(BF), torch.tensor([-1, 2, 5], device="cuda")
    for scale in (math.inf, math.nan):
        y = clusters.cluster_lookup(t, ids, scale=scale)
        assert y[0].eq(0).all() and y[2].eq(0).all() and not y[1].isfinite().any()
