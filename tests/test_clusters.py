"""CPU tests of the operators on clustered rows: the C-ABI checks every argument on the
host before any CUDA call, and the Python layer refuses tensors that are not on a GPU."""

from __future__ import annotations

import ctypes

import pytest
import torch

from flash_kmeans_cuda import _lib, clusters

L = _lib.lib


def desc(**kw):
    d = _lib.AttentionDesc()
    for name in ("q", "k", "v", "sel", "order", "offsets"):
        setattr(d, name, 4096)
    for name in ("q_stride", "k_stride", "v_stride"):
        setattr(d, name, (ctypes.c_int64 * 3)(4096, 512, 64))
    sizes = dict(batch=2, q_heads=8, kv_heads=2, n_queries=5, n_keys=100, n_clusters=10, top_k=4, head_dim=64)
    for name, val in {**sizes, "dtype": 1, "scale": 0.125, **kw}.items():
        setattr(d, name, (ctypes.c_int64 * 3)(*val) if isinstance(val, tuple) else val)
    return d


BAD_DESC = [
    (dict(batch=0), "must be >= 1"),
    (dict(top_k=0), "must be >= 1"),
    (dict(q_heads=7), "multiple of kv_heads"),
    (dict(dtype=2), "dtype"),
    (dict(dtype=9), "dtype"),
    (dict(head_dim=60), "head_dim"),
    (dict(head_dim=136), "head_dim"),
    (dict(n_queries=1 << 31), "int32"),
    (dict(top_k=1025), "top_k"),
    (dict(q=None), "non-null"),
    (dict(q=4104), "16-byte"),
    (dict(q_stride=(4096, 512, 60)), "16-byte"),
]


@pytest.mark.parametrize("kw,msg", BAD_DESC + [
    (dict(k=None), "non-null"),
    (dict(sel=None), "non-null"),
    (dict(order=None), "non-null"),
    (dict(v=4104), "16-byte"),
    (dict(k_stride=(4096, 4, 64)), "16-byte"),
    (dict(top_k=1024, n_keys=1 << 21), "2^30"),
])
def test_attention_refuses(kw, msg):
    d = desc(**kw)
    assert L.fkc_cluster_attention(ctypes.byref(d), 4096, 4096, None, 0, None) == -1
    assert msg in _lib.last_error()
    assert L.fkc_cluster_attention_grad(ctypes.byref(d), 4096, 4096, 4096, 4096, 4096, 4096, None, 0, None) == -1
    assert msg in _lib.last_error()
    assert L.fkc_cluster_attention_workspace_size(ctypes.byref(d)) == 0
    assert L.fkc_cluster_attention_grad_workspace_size(ctypes.byref(d)) == 0


@pytest.mark.parametrize("kw,msg", BAD_DESC + [
    (dict(n_clusters=16385), "16384"),
    (dict(q_pos=4096, order=None), "order"),
])
def test_select_refuses(kw, msg):
    d = desc(**kw)
    assert L.fkc_cluster_select(ctypes.byref(d), 4096, None, 4096, None, 0, None) == -1
    assert msg in _lib.last_error()


def test_attention_workspaces_and_outputs_are_checked():
    d = desc()
    assert L.fkc_cluster_attention(None, 4096, 4096, None, 0, None) == -1
    assert L.fkc_cluster_attention(ctypes.byref(d), None, 4096, None, 0, None) == -1
    assert L.fkc_cluster_attention(ctypes.byref(d), 4104, 4096, None, 0, None) == -1
    need = L.fkc_cluster_attention_grad_workspace_size(ctypes.byref(d))
    assert need > 0
    args = [4096] * 6
    assert L.fkc_cluster_attention_grad(ctypes.byref(d), *args, 4096, need - 1, None) == -5
    assert L.fkc_cluster_attention_grad(ctypes.byref(d), *args, 4100, need, None) == -1
    assert L.fkc_cluster_attention_grad(ctypes.byref(d), 4096, 4096, 4096, 4096, None, 4096, 4096, need, None) == -1
    assert "go together" in _lib.last_error()
    need = L.fkc_cluster_select_workspace_size(ctypes.byref(d))
    assert need >= 4 * 2 * 2 * 5 * 10
    assert L.fkc_cluster_select(ctypes.byref(d), 4096, None, 4096, 4096, need - 1, None) == -5
    assert L.fkc_cluster_select(ctypes.byref(d), 4104, None, 4096, 4096, need, None) == -1
    # few queries of long selections: the parts of the split keys need room
    d = desc(n_queries=1, n_keys=1 << 16, n_clusters=256, top_k=64)
    assert L.fkc_cluster_attention_workspace_size(ctypes.byref(d)) > 0
    assert L.fkc_cluster_attention(ctypes.byref(d), 4096, 4096, None, 0, None) == -5


@pytest.mark.parametrize("B,N,K", [(0, 1, 1), (1, 0, 1), (1, 1, 0), (1, 1 << 31, 1), (1, 1, 1 << 31), (1 << 21, 1, 1)])
def test_order_and_lookup_refuse_sizes(B, N, K):
    assert L.fkc_cluster_order(4096, 0, 4096, 4096, B, N, K, 4096, 1 << 40, None) == -1
    assert L.fkc_cluster_order_workspace_size(B, N, K) == 0
    assert L.fkc_cluster_lookup(4096, 4096, 0, 4096, B, N, K, 8, 0, 1.0, None) == -1
    assert L.fkc_cluster_lookup_grad(4096, 4096, 0, 4096, B, N, K, 8, 0, 1.0, 4096, 1 << 40, None) == -1
    assert L.fkc_cluster_lookup_grad_workspace_size(B, N, K, 8) == 0


def test_order_and_lookup_refuse_pointers():
    assert L.fkc_cluster_order(None, 0, 4096, 4096, 1, 8, 4, None, 0, None) == -1
    assert "non-null" in _lib.last_error()
    assert L.fkc_cluster_order(4100, 1, 4096, 4096, 1, 8, 4, None, 0, None) == -1
    assert "aligned" in _lib.last_error()
    need = L.fkc_cluster_order_workspace_size(2, 100000, 512)
    assert need > 0
    assert L.fkc_cluster_order(4096, 0, 4096, 4096, 2, 100000, 512, 4096, need - 1, None) == -5
    assert L.fkc_cluster_lookup(4096, None, 0, 4096, 1, 8, 4, 8, 0, 1.0, None) == -1
    assert L.fkc_cluster_lookup(4096, 4096, 0, 4096, 1, 8, 4, 8, 5, 1.0, None) == -1
    need = L.fkc_cluster_lookup_grad_workspace_size(1, 1000, 50, 8)
    assert need >= 4 * 1000
    assert L.fkc_cluster_lookup_grad(4096, 4096, 0, 4096, 1, 1000, 50, 8, 0, 1.0, 4096, need - 1, None) == -5


def test_good_arguments_pass_to_the_device_check():
    if torch.cuda.is_available():
        pytest.skip("host has a GPU")
    d = desc()
    assert L.fkc_cluster_attention(ctypes.byref(d), 4096, 4096, 4096, 1 << 30, None) == -3
    assert L.fkc_cluster_order(4096, 0, 4096, 4096, 1, 8, 4, 4096, 1 << 20, None) == -3


def test_cpu_tensors_are_refused():
    ids = torch.zeros(1, 4, dtype=torch.int32)
    t = torch.zeros(4, 8, dtype=torch.float16)
    q = torch.zeros(1, 1, 1, 8, dtype=torch.float16)
    with pytest.raises(ValueError, match="CUDA"):
        clusters.cluster_order(ids, 2)
    with pytest.raises(ValueError, match="CUDA"):
        clusters.cluster_lookup(t, ids)
    with pytest.raises(ValueError, match="CUDA"):
        clusters.cluster_select(q, t[None], ids, 2)
    with pytest.raises(ValueError, match="CUDA"):
        clusters.cluster_attention(q, q, q, ids[None], ids, ids)


def test_forward_mode_tangents_are_refused():
    """A dual tensor that does not require grad too: its tangent would be dropped, a derivative of zero."""
    t = torch.zeros(4, 8, dtype=torch.float16)
    q = torch.zeros(1, 1, 1, 8, dtype=torch.float16)
    ids = torch.zeros(1, 4, dtype=torch.int32)
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(RuntimeError, match="tangent"):
            clusters.cluster_lookup(torch.autograd.forward_ad.make_dual(t, t), ids)
        d = torch.autograd.forward_ad.make_dual(q, q)
        for args in ((d, q, q), (q, d, q), (q, q, d)):
            with pytest.raises(RuntimeError, match="tangent"):
                clusters.cluster_attention(*args, ids[None], ids, ids)


def test_selection_scratch_does_not_grow_with_the_prompt():
    for kw in (dict(n_queries=1 << 16, n_clusters=4096), dict(n_queries=1 << 16, n_clusters=16384),
               dict(batch=1 << 16, n_queries=3, n_clusters=16384), dict(n_queries=1 << 20, n_clusters=1)):
        need = L.fkc_cluster_select_workspace_size(ctypes.byref(desc(**kw)))
        assert 0 < need <= 160 << 20, (kw, need)


def test_attention_scratch_is_bounded():
    """Whatever the sizes: 4 GB of units' rows for out and 8 GB for the gradients, a quarter more with all."""
    for batch, kv, group, nq, n, clusters, top in [(1, 8, 4, 1 << 15, 1 << 15, 512, 16), (1, 8, 4, 1 << 17, 1 << 17, 2048, 64), (64, 8, 8, 4096, 8192, 128, 32),
                                                   (256, 8, 16, 64, 4096, 64, 64), (1024, 8, 4, 64, 2048, 1024, 16), (1, 1, 128, 1 << 15, 1 << 15, 64, 64)]:
        for head_dim in (64, 128):
            d = desc(batch=batch, q_heads=kv * group, kv_heads=kv, n_queries=nq, n_keys=n, n_clusters=clusters, top_k=top, head_dim=head_dim,
                     q_stride=(kv * group * nq * head_dim, nq * head_dim, head_dim), k_stride=(kv * n * head_dim, n * head_dim, head_dim),
                     v_stride=(kv * n * head_dim, n * head_dim, head_dim))
            assert L.fkc_cluster_attention_workspace_size(ctypes.byref(d)) <= 5 << 30
            assert L.fkc_cluster_attention_grad_workspace_size(ctypes.byref(d)) <= 10 << 30


def test_gradients_do_not_need_out():
    """out may be left out: the gradients sum what they need of it anew."""
    if torch.cuda.is_available():
        pytest.skip("host has a GPU")
    d = desc()
    need = L.fkc_cluster_attention_grad_workspace_size(ctypes.byref(d))
    assert L.fkc_cluster_attention_grad(ctypes.byref(d), None, 4096, 4096, 4096, 4096, 4096, 4096, need, None) == -3
    assert L.fkc_cluster_attention_grad(ctypes.byref(d), None, None, 4096, 4096, 4096, 4096, 4096, need, None) == -1
    assert "lse" in _lib.last_error()
