"""Plain 64-bit forms of the operators in ``flash_kmeans_cuda.clusters``, and how far a
16-bit kernel may be from them.

Tolerances count roundings: ``u = finfo(dtype).eps / 2`` for each value rounded to the
16-bit type, ``(terms) * 2**-22`` for sums on the tensor cores (each addition truncates at
2**-22 of the largest magnitude at worst).
"""

from __future__ import annotations

import math

import torch


def order_ref(ids, K):
    ids = ids.cpu().long()
    key = torch.where((ids < 0) | (ids >= K), K, ids)
    order = torch.sort(key, dim=1, stable=True).indices
    offsets = torch.stack([(key < k).sum(1) for k in range(K + 1)], 1) if K < 64 else \
        torch.searchsorted(key.sort(1).values, torch.arange(K + 1).repeat(ids.shape[0], 1).contiguous())
    slot = torch.arange(ids.shape[1])[None]
    return torch.where(slot < offsets[:, K:], order, -1).int(), offsets.int()


def reads(sel, order, offsets, q_pos, Hkv):
    """How often query i of row r reads key j: (R, Nq, N) float64."""
    R, Nq, top = sel.shape
    N, K = order.shape[1], offsets.shape[1] - 1
    m = torch.zeros(R, Nq, N, dtype=torch.float64, device=sel.device)
    for r in range(R):
        member = torch.zeros(K, N, dtype=torch.float64, device=sel.device)
        off = offsets[r].tolist()
        for c in range(K):
            rows = order[r, off[c]:off[c + 1]].long()
            member[c, rows[(rows >= 0) & (rows < N)]] = 1.0
        times = torch.zeros(Nq, K + 1, dtype=torch.float64, device=sel.device)
        ok = (sel[r] >= 0) & (sel[r] < K)
        times.scatter_add_(1, torch.where(ok, sel[r], K).long(), torch.ones(Nq, top, dtype=torch.float64, device=sel.device))
        m[r] = times[:, :K] @ member
        if q_pos is not None:
            m[r] *= torch.arange(N, device=sel.device)[None] <= q_pos[r // Hkv][:, None]
    return m


def attention_ref(q, k, v, sel, order, offsets, q_pos=None, scale=None, dout=None):
    """(values, tolerances): dicts with out, lse and, for a dout, dq, dk, dv; float64."""
    B, Hq, Nq, D = q.shape
    Hkv, N = k.shape[1], k.shape[2]
    G = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    u = torch.finfo(q.dtype).eps / 2
    m = reads(sel, order, offsets, q_pos, Hkv).view(B, Hkv, 1, Nq, N)
    seen = m > 0
    used = seen.any(3).any(2)  # keys that no query sees have no influence, whatever they hold
    qd = q.double().view(B, Hkv, G, Nq, D)
    alive = seen.any(-1).expand(B, Hkv, G, Nq)
    qd = torch.where(alive[..., None], qd, 0.0)
    kd = torch.where(used[..., None], k.double(), 0.0)[:, :, None]
    vd = torch.where(used[..., None], v.double(), 0.0)[:, :, None]
    s = qd @ kd.transpose(-1, -2) * scale
    top = s.masked_fill(~seen, -math.inf).amax(-1, keepdim=True)
    p = torch.where(seen, m * torch.exp(s - top.masked_fill(top == -math.inf, 0.0)), 0.0)
    l = p.sum(-1, keepdim=True)
    p = p / l.masked_fill(l == 0, 1.0)
    out = p @ vd
    lse = (top + l.log()).squeeze(-1)
    # the scores' error: products are exact, D additions; scale and exp2's argument round too
    mag = qd.norm(dim=-1, keepdim=True) * kd.norm(dim=-1)[..., None, :] * abs(scale)  # a magnitude: |scale|, whatever its sign
    mag = torch.where(seen, mag, 0.0).amax(-1, keepdim=True)
    ds_ = mag * (D + 8) * 2.0 ** -22 + 2.0 ** -20  # relative error of a weight, numerator ...
    rel = 4 * ds_                                   # ... and the sum, with room for the square
    n_add = min(N, int(m.sum(-1).max().item()) if m.numel() else 1) + 8
    acc = n_add * 2.0 ** -22
    # the parts of a row over single clusters, which add up to p @ |v| at most in magnitude, may be
    # held with 11 bits (fp16 under a power of two) when out has 8: another 2**-11 of them
    held = 2.0 ** -11 if q.dtype == torch.bfloat16 else 0.0
    tol_out = (u + held + rel + acc) * (p @ vd.abs()) * (1 + u) + u * out.abs()
    val = {"out": out.reshape(q.shape), "lse": lse.reshape(B, Hq, Nq)}
    tol = {"out": tol_out.reshape(q.shape),
           "lse": (rel.squeeze(-1) + acc + 2.0 ** -22 * lse.abs().masked_fill(lse.isinf(), 0.0)).reshape(B, Hq, Nq)}
    if dout is not None:
        do = torch.where(alive[..., None], dout.double().view(B, Hkv, G, Nq, D), 0.0)
        dp = do @ vd.transpose(-1, -2)
        delta = (do * out).sum(-1, keepdim=True)
        ds = p * (dp - delta)
        val["dq"] = (ds @ kd * scale).reshape(q.shape)
        val["dk"] = (ds.transpose(-1, -2) @ qd * scale).sum(2)
        val["dv"] = (p.transpose(-1, -2) @ do).sum(2)
        # the kernel's delta comes from the rounded out; dP is D additions on the tensor cores
        e_delta = (do.abs() * tol_out).sum(-1, keepdim=True) + D * 2.0 ** -22 * (do * out).abs().sum(-1, keepdim=True)
        e_dp = (D + 8) * 2.0 ** -22 * (do.abs() @ vd.abs().transpose(-1, -2))
        e_ds = (u + rel) * ds.abs() + p * (e_delta + e_dp) * (1 + u + rel)
        cols = G * Nq + 8
        tol["dq"] = ((e_ds + acc * ds.abs()) @ kd.abs() * abs(scale)).reshape(q.shape) + u * val["dq"].abs()
        tol["dk"] = ((e_ds + cols * 2.0 ** -22 * ds.abs()).transpose(-1, -2) @ qd.abs() * abs(scale)).sum(2) + u * val["dk"].abs()
        tol["dv"] = (((u + rel + cols * 2.0 ** -22) * p).transpose(-1, -2) @ do.abs()).sum(2) + u * val["dv"].abs()
    tiny = {torch.float16: 2.0 ** -24, torch.bfloat16: 2.0 ** -126}[q.dtype]  # subnormal steps
    for name in tol:
        tol[name] = tol[name] + tiny * (1 if name in ("out", "lse") else 64)
    return val, tol


def select_ref(q, centroids, offsets, top, order=None, q_pos=None, bias=None, scale=None):
    B, Hq, Nq, D = q.shape
    R, K = centroids.shape[:2]
    Hkv = R // B
    scale = D ** -0.5 if scale is None else scale
    qd = q.double().view(R, Hq // Hkv, Nq, D)
    s = (qd[:, :, :, None, :] * centroids.double()[:, None, None]).sum(-1).amax(1) * scale  # amax keeps NaN
    if bias is not None:
        s = s + bias.double()[:, None]
    bad = ((offsets[:, 1:] - offsets[:, :-1]) <= 0)[:, None].expand(R, Nq, K)
    if q_pos is not None:
        first = order.gather(1, offsets[:, :-1].long().clamp(max=order.shape[1] - 1))
        bad = bad | (first[:, None] > q_pos.repeat_interleave(Hkv, 0)[:, :, None])
    s = torch.where(bad | s.isnan(), -math.inf, s)
    val, idx = torch.sort(s, dim=-1, descending=True, stable=True)
    idx = torch.where(val == -math.inf, K, idx)[..., :top].sort(-1).values
    idx = torch.where(idx == K, -1, idx)
    return torch.nn.functional.pad(idx, (0, top - idx.shape[-1]), value=-1).int()
