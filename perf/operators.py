"""The operators of ``flash_kmeans_cuda.clusters`` as measurable cases: grouping of
positions by cluster, lookup of centroids with its gradient, selection of clusters for a
query and attention over the keys of the selected clusters.

``listed`` and ``draw`` give cases, ``prepare`` makes a case's inputs on the GPU, ``run``
is one pass: the plain form in elementary torch operations, or, where ``own`` is true, the
package's calls. ``exact`` is the definition in 64 bits.

Shapes: ``batch`` sequences with ``hkv`` heads of keys (rows of clusters: ``batch * hkv``)
and ``group`` query heads for each of them.
"""

from __future__ import annotations

import math
import os
import sys

import torch

# the package's folder: its name is no module name
_PACKAGE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-kmeans-cuda_b200")
if _PACKAGE not in sys.path:
    sys.path.insert(0, _PACKAGE)

own = False

_TYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # grouping the keys of one layer's cache (8 heads) after they were clustered
        {"name": "order-layer", "op": "order", "rows": 8, "n": 32768, "k": 512},
        # the smallest grouping: one short prompt
        {"name": "order-short", "op": "order", "rows": 4, "n": 1000, "k": 20},
        # codes of one short sequence read back from a codebook: latency
        {"name": "lookup-short", "op": "lookup", "rows": 0, "n": 333, "k": 512, "d": 128, "type": "bf16", "scale": 1.0, "train": False},
        # a training step of a token embedding: ids of skewed frequency, scaled by sqrt(D)
        {"name": "lookup-embedding-train", "op": "lookup", "rows": 0, "n": 16384, "k": 50000, "d": 1024, "type": "bf16", "scale": 32.0, "train": True},
        # per-row codebooks of the batched benchmark shape (32 x 16384 rows of 64, 1024 clusters), trained in fp32
        {"name": "lookup-codebooks-train", "op": "lookup", "rows": 32, "n": 16384, "k": 1024, "d": 64, "type": "fp32", "scale": 1.0, "train": True},
        # one new token of each of 16 sequences chooses among 1024 clusters
        {"name": "select-decode", "op": "select", "batch": 16, "hkv": 8, "group": 4, "nq": 1, "n": 32768, "k": 1024, "d": 128, "type": "bf16", "top": 64, "causal": False},
        # every position of a prompt's last part chooses
        {"name": "select-prefill", "op": "select", "batch": 1, "hkv": 8, "group": 4, "nq": 4096, "n": 16384, "k": 256, "d": 128, "type": "bf16", "top": 16, "causal": True},
        # one token, one short sequence: latency
        {"name": "attend-decode-one", "op": "attend", "batch": 1, "hkv": 2, "group": 4, "nq": 1, "n": 4093, "k": 64, "d": 64, "type": "fp16", "top": 8, "causal": True, "train": False},
        # a batch of single tokens over long caches: the bytes of the selected keys
        {"name": "attend-decode-batch", "op": "attend", "batch": 16, "hkv": 8, "group": 4, "nq": 1, "n": 32768, "k": 1024, "d": 128, "type": "bf16", "top": 64, "causal": True, "train": False},
        # the last 4096 positions of a prompt of 16384
        {"name": "attend-prefill", "op": "attend", "batch": 1, "hkv": 8, "group": 4, "nq": 4096, "n": 16384, "k": 256, "d": 128, "type": "bf16", "top": 16, "causal": True, "train": False},
        # a training step of one layer over a sequence of 4096
        {"name": "attend-train", "op": "attend", "batch": 1, "hkv": 4, "group": 4, "nq": 4096, "n": 4096, "k": 64, "d": 128, "type": "bf16", "top": 8, "causal": True, "train": True},
        # a small padded batch with odd sizes: a head size between the tiles, three heads a group
        {"name": "attend-train-odd", "op": "attend", "batch": 2, "hkv": 2, "group": 3, "nq": 777, "n": 777, "k": 13, "d": 80, "type": "fp16", "top": 5, "causal": True, "train": True},
    ]


def _spread(rng, low, high):
    """A whole number between low and high, spread over the logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["order", "lookup", "select", "attend", "attend"])
    if op == "order":
        rows = rng.randint(1, 16)
        n = _spread(rng, 16, 524288 // rows)
        return {"op": op, "rows": rows, "n": n, "k": _spread(rng, 2, 8192)}
    if op == "lookup":
        train = rng.random() < 0.6
        if rng.random() < 0.5:
            rows, d = 0, 8 * _spread(rng, 2, 256)
            n, k = _spread(rng, 1, 16384), _spread(rng, 2, max(2, min(65536, 50_000_000 // d)))
        else:
            rows, d = rng.randint(1, 32), 16 * rng.randint(1, 8)
            n, k = _spread(rng, 1, 16384), _spread(rng, 2, 2048)
        return {"op": op, "rows": rows, "n": n, "k": k, "d": d, "type": rng.choice(["bf16", "fp16", "fp32"]),
                "scale": rng.choice([1.0, 0.125, math.sqrt(d)]), "train": train}
    c = {"op": op, "batch": rng.randint(1, 4), "hkv": rng.choice([1, 2, 4, 8]), "group": rng.choice([1, 2, 3, 4, 5, 8, 16]),
         "d": rng.choice([32, 64, 80, 96, 112, 128]), "type": rng.choice(["bf16", "fp16"]), "causal": rng.random() < 0.7}
    heads = c["batch"] * c["hkv"] * c["group"]
    decode = rng.random() < 0.4
    c["n"] = _spread(rng, 16 if op == "attend" else 1024, 32768 if decode else 4096)
    c["nq"] = rng.randint(1, 2) if decode else min(c["n"], _spread(rng, 1, max(2, 400_000_000 // (heads * c["n"]))))
    c["k"] = max(1, c["n"] // rng.choice([16, 32, 64, 100]))
    c["top"] = rng.randint(1, min(64, c["k"] if op == "attend" else c["k"] // 2))
    if op == "attend":
        c["train"] = not decode and rng.random() < 0.5
    return c


# ---------------------------------------------------------------------------- inputs
def _labels(rows, n, k, gen):
    """Cluster ids of skewed sizes: the density falls with the rank's cube root, the ranks are shuffled."""
    rank = (k * torch.rand(rows, n, generator=gen, device="cuda") ** 1.5).long().clamp(max=k - 1)
    return torch.rand(rows, k, generator=gen, device="cuda").argsort(1).gather(1, rank).to(torch.int32)


def _group(ids, k):
    """What cluster_order gives: positions by cluster, and each cluster's first slot. ids of -1 come last, as -1."""
    key = torch.where(ids < 0, k, ids).long()
    order = torch.sort(key, dim=1, stable=True).indices.to(torch.int32)
    count = torch.zeros(ids.shape[0], k + 1, dtype=torch.long, device=ids.device)
    count.scatter_add_(1, key, torch.ones_like(key))
    offsets = torch.zeros(ids.shape[0], k + 1, dtype=torch.int32, device=ids.device)
    offsets[:, 1:] = count[:, :k].cumsum(1).to(torch.int32)
    slot = torch.arange(ids.shape[1], device=ids.device)
    order = torch.where(slot[None] < offsets[:, -1:], order, -1)
    return order.contiguous(), offsets


def _scores(q, centroids, size, first, q_pos, scale):
    """Exact scores (rows, Nq, K) of the clusters for each query: the group's best head, plus log of the size."""
    batch, hq, nq, d = q.shape
    rows = centroids.shape[0]
    qr = q.double().reshape(rows, -1, nq, d)
    s = (qr @ centroids.double()[:, None].transpose(-1, -2)).amax(1) * scale
    s = s + size.double().log().float().double()[:, None, :]
    out = size[:, None, :] == 0
    if q_pos is not None:
        out = out | (first[:, None, :] > q_pos.repeat_interleave(rows // batch, 0)[:, :, None])
    return s.masked_fill(out, -math.inf)


def _best(s, top):
    """The `top` best of the last dimension, ties to the lowest index; ascending, -1 behind them."""
    k = s.shape[-1]
    val, idx = torch.sort(s, dim=-1, descending=True, stable=True)
    val, idx = val[..., :top], idx[..., :top]
    idx = torch.where(val == -math.inf, k, idx).sort(-1).values
    idx = torch.where(idx == k, -1, idx).to(torch.int32)
    pad = top - idx.shape[-1]
    return torch.nn.functional.pad(idx, (0, pad), value=-1).contiguous()


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(1000 + seed)
    st = {"case": case}
    if case["op"] == "order":
        st["ids"] = _labels(case["rows"], case["n"], case["k"], gen)
        return st
    t, d, n, k = _TYPES[case["type"]], case["d"], case["n"], case["k"]

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    if case["op"] == "lookup":
        rows = case["rows"]
        if rows == 0:  # one table of tokens: frequencies fall as 1 / rank, the ranks are shuffled
            rank = (k ** torch.rand(n, generator=gen, device="cuda")).long().clamp(1, k) - 1
            st["table"] = normal(k, d).to(t)
            st["ids"] = torch.randperm(k, generator=gen, device="cuda")[rank].to(torch.int32)
        else:
            st["table"], st["ids"] = normal(rows, k, d).to(t), _labels(rows, n, k, gen)
        if case["train"]:
            st["table"].requires_grad_(True)
            st["dy"] = normal(*st["ids"].shape, d).to(t)
        return st
    batch, hkv, nq = case["batch"], case["hkv"], case["nq"]
    rows, hq = batch * hkv, hkv * case["group"]
    ids = _labels(rows, n, k, gen)
    key = torch.empty(rows, n, d, device="cuda", dtype=t)
    centre = normal(rows, k, d)
    key.copy_(centre.gather(1, ids.long()[..., None].expand(-1, -1, d)) + 0.5 * normal(rows, n, d))
    if case["causal"] and batch > 1 and n > 64:  # a padded batch: the odd sequences are a little shorter
        ids = ids.view(batch, hkv, n).clone()
        ids[1::2, :, n - n // 10:] = -1
        ids = ids.view(rows, n)
    st["order"], st["offsets"] = _group(ids, k)
    size = (st["offsets"][:, 1:] - st["offsets"][:, :-1])
    st["centroids"] = centre.to(t)
    st["bias"] = size.double().log().float()
    st["q"] = normal(batch, hq, nq, d).to(t)
    st["q_pos"] = None
    if case["causal"]:
        pos = torch.arange(n - nq, n, device="cuda", dtype=torch.int32).repeat(batch, 1)
        if batch > 1 and n > 64:
            pos[1::2] = torch.where(pos[1::2] >= n - n // 10, -1, pos[1::2]) if nq > 2 else n - n // 10 - 1
        st["q_pos"] = pos
    if case["op"] == "attend":
        first = _first(st["order"], st["offsets"])
        st["sel"] = _best(_scores(st["q"], st["centroids"], size, first, st["q_pos"], d ** -0.5), case["top"])
        st["k"], st["v"] = key.view(batch, hkv, n, d), normal(batch, hkv, n, d).to(t)
        if case["train"]:
            for name in ("q", "k", "v"):
                st[name].requires_grad_(True)
            st["dout"] = normal(batch, hq, nq, d).to(t)
    return st


def _first(order, offsets):
    """The first position of each cluster (rows, K): what an empty cluster has is of no account."""
    at = offsets[:, :-1].long().clamp(max=order.shape[1] - 1)
    return order.gather(1, at)


# ---------------------------------------------------------------------------- the passes
def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"order": _order, "lookup": _lookup, "select": _select, "attend": _attend}[state["case"]["op"]](state)


def _run_own(state):
    from flash_kmeans_cuda import clusters

    case = state["case"]
    if case["op"] == "order":
        return clusters.cluster_order(state["ids"], case["k"])
    if case["op"] == "lookup":
        y = clusters.cluster_lookup(state["table"], state["ids"], scale=case["scale"])
        if not case["train"]:
            return y
        return y.detach(), torch.autograd.grad(y, state["table"], state["dy"])[0]
    if case["op"] == "select":
        return clusters.cluster_select(state["q"], state["centroids"], state["offsets"], case["top"],
                                       order=state["order"], q_pos=state["q_pos"], bias=state["bias"])
    args = [state[name] for name in ("q", "k", "v", "sel", "order", "offsets")]
    if not case["train"]:
        return clusters.cluster_attention(*args, q_pos=state["q_pos"], return_lse=True)
    out = clusters.cluster_attention(*args, q_pos=state["q_pos"])
    return (out.detach(), *torch.autograd.grad(out, args[:3], state["dout"]))


def _order(st):
    return _group(st["ids"], st["case"]["k"])


def _lookup(st):
    table, ids, scale = st["table"], st["ids"], st["case"]["scale"]
    flat = table.reshape(-1, table.shape[-1]).float()
    at = ids.long() if table.dim() == 2 else ids.long() + torch.arange(table.shape[0], device="cuda")[:, None] * table.shape[1]
    y = (flat[at] * scale).to(table.dtype)
    if not st["case"]["train"]:
        return y
    grad = torch.zeros_like(flat).index_add_(0, at.reshape(-1), st["dy"].float().reshape(-1, flat.shape[1]))
    return y, (grad * scale).to(table.dtype).view(table.shape)


def _select(st):
    # in 64 bits: the border between the last chosen cluster and the next is a comparison
    size = st["offsets"][:, 1:] - st["offsets"][:, :-1]
    scale = st["case"]["d"] ** -0.5
    s = _scores(st["q"], st["centroids"], size, _first(st["order"], st["offsets"]), st["q_pos"], scale)
    return _best(s, st["case"]["top"])


def _attend(st):
    q, k, v, sel, order, offsets = (st[name] for name in ("q", "k", "v", "sel", "order", "offsets"))
    batch, hq, nq, d = q.shape
    rows, n = order.shape
    hkv, kc = rows // batch, offsets.shape[1] - 1
    scale = d ** -0.5
    # how often query i reads key j: what it selected, looked up at the key's cluster
    slot = torch.arange(n, device="cuda", dtype=torch.int32).repeat(rows, 1)
    of_slot = torch.searchsorted(offsets[:, 1:].contiguous(), slot, right=True)
    valid = order >= 0
    label = torch.full((rows, n + 1), kc, device="cuda").scatter_(1, torch.where(valid, order, n).long(), of_slot.clamp(max=kc))[:, :n]
    times = torch.zeros(rows, nq, kc + 2, device="cuda").scatter_add_(2, torch.where(sel < 0, kc + 1, sel).long(), torch.ones(sel.shape, device="cuda"))
    reads = times[:, :, :kc + 1].gather(2, label[:, None].expand(-1, nq, -1))
    if st["q_pos"] is not None:
        late = torch.arange(n, device="cuda")[None, None] > st["q_pos"][:, :, None]
        reads = reads.masked_fill(late.repeat_interleave(hkv, 0), 0.0)
    reads = reads[:, None]  # rows, 1, nq, n
    qr, kr, vr = q.float().reshape(rows, -1, nq, d), k.float().reshape(rows, 1, n, d), v.float().reshape(rows, 1, n, d)
    s = qr @ kr.transpose(-1, -2) * scale
    top = s.masked_fill(reads == 0, -math.inf).amax(-1, keepdim=True)
    p = torch.where(reads == 0, 0.0, reads * torch.exp(s - torch.where(top == -math.inf, 0.0, top)))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total == 0, 1.0, total)
    out = p @ vr
    o = out.reshape(q.shape).to(q.dtype)
    if not st["case"]["train"]:
        return o, (top + torch.log(total)).reshape(batch, hq, nq)
    do = st["dout"].float().reshape(rows, -1, nq, d)
    ds = p * (do @ vr.transpose(-1, -2) - (do * out).sum(-1, keepdim=True)) * scale
    dq = ds @ kr
    dk, dv = (ds.transpose(-1, -2) @ qr).sum(1), (p.transpose(-1, -2) @ do).sum(1)
    return o, dq.reshape(q.shape).to(q.dtype), dk.reshape(k.shape).to(k.dtype), dv.reshape(v.shape).to(v.dtype)


# ---------------------------------------------------------------------------- sizes and the definition
def work(case):
    if case["op"] == "order":
        return {"bytes": 4 * case["rows"] * (2 * case["n"] + case["k"] + 1), "flops": 0}
    s, d, n, k = _BYTES[case["type"]], case["d"], case["n"], case["k"]
    if case["op"] == "lookup":
        rows = max(1, case["rows"])
        entries = rows * n
        read = min(entries, rows * k)  # rows of the table, each once
        b = 4 * entries + s * d * (read + entries)
        f = entries * d
        if case["train"]:
            b += s * d * (entries + rows * k)
            f += 2 * entries * d
        return {"bytes": b, "flops": f}
    rows, nq = case["batch"] * case["hkv"], case["nq"]
    heads = rows * case["group"]
    if case["op"] == "select":
        return {"bytes": s * d * (heads * nq + rows * k) + 4 * rows * (2 * k + 1 + nq * case["top"]), "flops": 2 * heads * nq * k * d}
    seen = min(1.0, case["top"] / k) * n  # keys in the selected clusters of one query
    part = (n - 0.5 * (nq - 1)) / n if case["causal"] else 1.0  # of which it may see
    touched = min(n, nq * seen)
    b = s * d * (2 * heads * nq + 2 * rows * touched) + 4 * rows * (touched + nq * case["top"] + k + 1) + 4 * heads * nq
    f = 4 * heads * nq * seen * part * d
    if case["train"]:
        b += s * d * (2 * heads * nq + 2 * rows * n)
        f += 10 * heads * nq * seen * part * d
    return {"bytes": int(b), "flops": int(f)}


@torch.no_grad()
def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] in ("order", "select"):
        return None  # whole numbers
    if case["op"] == "lookup":
        table, ids = st["table"].double(), st["ids"].long()
        three = table if table.dim() == 3 else table[None]
        two = ids.reshape(three.shape[0], -1)
        y = torch.stack([three[b].index_select(0, two[b]) for b in range(three.shape[0])]) * case["scale"]
        y = y.reshape(*ids.shape, table.shape[-1])
        if not case["train"]:
            return y
        dy = st["dy"].double().reshape(three.shape[0], -1, table.shape[-1])
        g = torch.stack([torch.zeros_like(three[b]).index_add_(0, two[b], dy[b]) for b in range(three.shape[0])]) * case["scale"]
        return y, g.reshape(table.shape)
    q, k, v, sel, order, offsets = (st[name] for name in ("q", "k", "v", "sel", "order", "offsets"))
    batch, hq, nq, d = q.shape
    rows, n = order.shape
    hkv, group = rows // batch, hq // (rows // batch)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    lse = torch.full(q.shape[:3], -math.inf, dtype=torch.float64, device="cuda")
    dq, dk, dv = torch.zeros_like(out), torch.zeros(k.shape, dtype=torch.float64, device="cuda"), torch.zeros(v.shape, dtype=torch.float64, device="cuda")
    for r in range(rows):
        b, h = divmod(r, hkv)
        heads = slice(h * group, (h + 1) * group)
        used = int(offsets[r, -1])
        at = order[r, :used].long()  # keys in cluster order
        size = (offsets[r, 1:] - offsets[r, :-1]).long()
        of = torch.repeat_interleave(torch.arange(size.numel(), device="cuda"), size)
        listed_times = (sel[r][:, :, None] == torch.arange(size.numel(), device="cuda", dtype=torch.int32)).sum(1).double()
        weight = listed_times[:, of]
        if st["q_pos"] is not None:
            weight = weight * (at[None] <= st["q_pos"][b][:, None])
        kk, vv = k[b, h, at].double(), v[b, h, at].double()
        for head in range(heads.start, heads.stop):
            z = q[b, head].double() @ kk.T * d ** -0.5 + weight.log()
            m = torch.logsumexp(z, -1) if used else torch.full((nq,), -math.inf, dtype=torch.float64, device="cuda")
            p = torch.exp(z - m[:, None].masked_fill(m[:, None] == -math.inf, 0.0))
            lse[b, head], o = m, p @ vv
            out[b, head] = o
            if case["train"]:
                do = st["dout"][b, head].double()
                dz = p * (do @ vv.T - (do * o).sum(1)[:, None]) * d ** -0.5
                dq[b, head] = dz @ kk
                dk[b, h].index_add_(0, at, dz.T @ q[b, head].double())
                dv[b, h].index_add_(0, at, p.T @ do)
    return (out, dq, dk, dv) if case["train"] else (out, lse)
