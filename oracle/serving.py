"""Plain 64-bit forms of the batched-serving operators (kv_slots, qk_norm_rope_kv_paged, tree_attention, sample_next):
the definitions in include/lfm2q.h written out on the CPU, one request, head or row at a time."""

import math

import numpy as np
import torch


def kv_slots_ref(lens, new_lens, table, free, n_free, page, capacity):
    """Returns (got, cu, positions, slots, table, free, n_free) as numpy arrays / an int; positions and slots hold the
    granted tokens only. Inputs are numpy integer arrays and are not changed."""
    table, free = table.copy(), free.copy()
    B, width = table.shape
    room = width * page
    got, cu, positions, slots, grown, shrunk = [], [0], [], [], [], []
    pages_sum = tokens_sum = 0
    for b in range(B):
        l, w = int(lens[b]), int(new_lens[b])
        ok = 0 <= l <= room and 0 <= w <= room
        pl, pw = -(-l // page), -(-w // page)
        if ok:
            pages_sum += max(0, pw - pl)
            tokens_sum += max(0, w - l)
            ok = (pw <= pl or pages_sum <= n_free) and (w <= l or tokens_sum <= capacity)
        got.append(w if ok else l)
        cu.append(cu[-1] + (max(0, w - l) if ok else 0))
        if ok:
            for j in range(pl, pw):
                table[b, j] = free[n_free - 1 - len(grown)]
                grown.append((b, j))
            shrunk += [(b, j) for j in range(pw, pl)]
            for t in range(l, w):
                positions.append(t)
                slots.append(int(table[b, t // page]) * page + t % page)
    top = n_free - len(grown) + len(shrunk)
    for i, (b, j) in enumerate(shrunk):
        free[top - 1 - i] = table[b, j]
        table[b, j] = -1
    return (np.array(got), np.array(cu), np.array(positions, np.int64), np.array(slots, np.int64), table, free, top)


def rope_paged_f64(qkv, qw, kw, inv_freq, scaling, positions, slots, kc, vc, NQ, eps, interleaved):
    """(q [N, NQ, D], kc, vc) in fp64 (CPU tensors; the caches come back with the new rows in them)."""
    pages, NKV, page, D = kc.shape
    N, R = qkv.shape[0], 2 * inv_freq.numel()
    x = qkv.double().view(N, NQ + 2 * NKV, D)
    kc, vc = kc.double().clone(), vc.double().clone()
    q = torch.empty(N, NQ, D, dtype=torch.float64)
    for n in range(N):
        ang = [float(positions[n]) * float(f) for f in inv_freq.double()]
        c = torch.tensor([math.cos(a) * scaling for a in ang], dtype=torch.float64)
        s = torch.tensor([math.sin(a) * scaling for a in ang], dtype=torch.float64)
        for h in range(NQ + NKV):
            v = x[n, h].clone()
            w = qw if h < NQ else kw
            if w is not None:
                v = v / torch.sqrt((v * v).mean() + eps) * w.double()
            i = torch.arange(R // 2)
            a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
            va, vb = v[a].clone(), v[b].clone()
            v[a] = va * c - vb * s
            v[b] = vb * c + va * s
            if h < NQ:
                q[n, h] = v
            elif 0 <= int(slots[n]) < pages * page:
                kc[int(slots[n]) // page, h - NQ, int(slots[n]) % page] = v
        if 0 <= int(slots[n]) < pages * page:
            vc[int(slots[n]) // page, :, int(slots[n]) % page] = x[n, NQ + NKV:]
    return q, kc, vc


def tree_attention_f64(q, kc, vc, table, ctx, cu, mask, scale, max_q=64):
    """[N, NQ, D] in fp64; rows outside the requests (or past max_q of one) are NaN. mask: [N] Python ints or None."""
    N, NQ, D = q.shape
    pages, NKV, page, _ = kc.shape
    G, room = NQ // NKV, table.shape[1] * page
    out = torch.full((N, NQ, D), float("nan"), dtype=torch.float64)
    for b in range(len(ctx)):
        n0 = int(cu[b])
        T = min(int(cu[b + 1]) - n0, max_q)
        c = int(ctx[b])
        L = min(c + T, room)
        pid = [int(table[b, t // page]) for t in range(L)]
        live = [0 <= p < pages for p in pid]
        rows = [(p * page + t % page) if ok else 0 for t, (p, ok) in enumerate(zip(pid, live))]
        for i in range(T):
            m = (2 << i) - 1 if mask is None else int(mask[n0 + i])
            see = [t for t in range(L) if live[t] and (t < c or (m >> (t - c)) & 1)]
            idx = torch.tensor([rows[t] for t in see], dtype=torch.long)
            for h in range(NKV):
                k = kc[:, h].reshape(-1, D)[idx].double()
                v = vc[:, h].reshape(-1, D)[idx].double()
                for g in range(G):
                    if not see:
                        out[n0 + i, h * G + g] = 0
                        continue
                    s = k @ q[n0 + i, h * G + g].double() * scale
                    p = torch.exp(s - s.max())
                    out[n0 + i, h * G + g] = (p @ v) / p.sum()
    return out


def sample_next_f64(logits, temperature, top_k, top_p, min_p, u):
    """The token of one row: logits a numpy array (any float type), the rest Python numbers. Masses are counted in whole
    steps of 2^-44 of the largest weight, as the operator defines them (a weight below half a step counts as none: only a
    u of 1 or more, held to the last step of the mass, would tell)."""
    x = np.asarray(logits, np.float64)
    if np.isnan(x).any():
        return int(np.flatnonzero(np.isnan(x))[0])
    if not temperature > 0 or x.max() == -np.inf:
        return int(np.argmax(x))
    order = np.lexsort((np.arange(len(x)), -x))
    if top_k > 0:
        order = order[:top_k]
    with np.errstate(invalid="ignore", over="ignore"):
        w = np.where(x == x.max(), 1.0, np.exp((x - x.max()) / temperature))
    w[x == -np.inf] = 0.0
    least = min(min_p, 1.0) if min_p > 0 else 0.0
    high, w = w >= least, np.rint(w * 2.0 ** 44)
    if top_p < 1:
        mass = w[order]
        before = np.cumsum(mass) - mass
        keep = before < max(top_p, 0.0) * mass.sum()
        keep[0] = True
        order = order[keep]
    order = np.sort(order[high[order]])
    run = np.cumsum(w[order])
    u = min(max(u, 0.0), 1.0) if u == u else 0.0
    return int(order[min(np.searchsorted(run, u * run[-1], side="right"), np.flatnonzero(w[order])[-1])])
