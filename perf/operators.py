"""What the batched-serving operators cost: block tables and slot maps (kv_slots), rotary positions into a paged cache
(qk_norm_rope_kv_paged), attention of a tree of drafted tokens over that cache (tree_attention) and sampling
(sample_next), each as elementary torch operations and as the framework's kernel.

`listed()` names the cases, `draw(rng)` makes more of the same ranges, `prepare` makes a case's inputs, `run` makes one
pass, `exact` gives the outputs from the definition in 64 bits and `work` the bytes and operations of one pass.
"""

import math
import sys
from pathlib import Path

import numpy as np
import torch

own = False

_PKG = Path(__file__).resolve().parents[1] / "lfm2.5-vl-optimization_b200"
_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_DEV = "cuda"


def _ext():
    if str(_PKG) not in sys.path:
        sys.path.insert(0, str(_PKG))
    from lfm2opt.kernels import ext
    return ext()


# ---------------------------------------------------------------------------------------------------- cases
def listed():
    return [
        # 37 chat requests that each draft 16 tokens on small pages, then give the pages back: latency
        {"name": "slots-draft-37x16", "op": "slots", "B": 37, "page": 16, "lo": 0, "hi": 8191, "add": 16,
         "spare": 100},
        # admission of 64 prompts of 1024 tokens (a 64 K token prefill batch)
        {"name": "slots-admit-64x1024", "op": "slots", "B": 64, "page": 64, "lo": 0, "hi": 0, "add": 1024,
         "spare": 1100},
        # one token of one request: LFM2's heads, q/k norm, half layout
        {"name": "rope-1", "op": "rope", "N": 1, "NQ": 32, "NKV": 8, "D": 64, "rot": 64, "interleaved": False,
         "norm": True, "dtype": "bf16", "page": 64, "far": 4000},
        # 300 drafted tokens of a batch, half of the head rotated, ragged count
        {"name": "rope-300-partial", "op": "rope", "N": 300, "NQ": 32, "NKV": 8, "D": 64, "rot": 32,
         "interleaved": False, "norm": False, "dtype": "bf16", "page": 16, "far": 32768},
        # a long-context prefill: interleaved layout, 128-wide heads, far positions
        {"name": "rope-16384-interleaved", "op": "rope", "N": 16384, "NQ": 32, "NKV": 8, "D": 128, "rot": 128,
         "interleaved": True, "norm": True, "dtype": "fp16", "page": 64, "far": 1000000},
        # one token of one request over 1001 positions: the paged form of the batch-1 decode step
        {"name": "tree-1x1", "op": "tree", "B": 1, "T": 1, "NQ": 32, "NKV": 8, "D": 64, "page": 64, "lo": 1000,
         "hi": 1000, "dtype": "bf16", "chain": True},
        # 13 drafted tokens of 5 requests on 128-wide heads and small pages, one of them with an empty cache
        {"name": "tree-5x13-wide", "op": "tree", "B": 5, "T": 13, "NQ": 24, "NKV": 3, "D": 128, "page": 16, "lo": 0,
         "hi": 777, "dtype": "fp16", "chain": False},
        # 32 requests with 16 drafted tokens each over chats of 500 to 4000 tokens
        {"name": "tree-32x16", "op": "tree", "B": 32, "T": 16, "NQ": 32, "NKV": 8, "D": 64, "page": 64, "lo": 500,
         "hi": 4000, "dtype": "bf16", "chain": False},
        # 16 requests with 64 drafted tokens each over long documents
        {"name": "tree-16x64-long", "op": "tree", "B": 16, "T": 64, "NQ": 32, "NKV": 8, "D": 64, "page": 64,
         "lo": 8000, "hi": 32000, "dtype": "bf16", "chain": False},
        # one request's next token, all filters on: latency
        {"name": "sample-1", "op": "sample", "B": 1, "V": 65536, "dtype": "bf16", "temp": 0.7, "k": 50, "p": 0.9,
         "minp": 0.05},
        # 64 requests with top-k and nucleus over an odd vocabulary (rows not aligned to 16 bytes)
        {"name": "sample-64-topk", "op": "sample", "B": 64, "V": 50001, "dtype": "bf16", "temp": 0.8, "k": 100,
         "p": 0.95, "minp": 0.0},
        # a large batch without top-k (the nucleus alone), logits in 32 bits
        {"name": "sample-256-nucleus", "op": "sample", "B": 256, "V": 65536, "dtype": "fp32", "temp": 1.0, "k": 0,
         "p": 0.95, "minp": 0.0},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["slots", "rope", "tree", "sample"])
    if op == "slots":
        B, page = _log(rng, 1, 256), rng.choice([1, 16, 24, 64, 128])
        hi = rng.randint(0, 8191 if page >= 16 else 700)
        add = _log(rng, 1, min(1024, (49152 if page > 1 else 24576) // B))
        need = B * (-(-add // page) + 1)
        spare = rng.choice([need, need, max(1, need // 2)])  # sometimes too few pages for all
        return {"op": op, "B": B, "page": page, "lo": hi // 3, "hi": hi, "add": add, "spare": spare}
    if op == "rope":
        D = rng.choice([64, 128])
        NKV = rng.randint(1, 8)
        return {"op": op, "N": _log(rng, 1, 16384), "NQ": NKV * rng.randint(1, 4), "NKV": NKV, "D": D,
                "rot": rng.choice([D, D, D // 2, 16]), "interleaved": rng.random() < 0.5, "norm": rng.random() < 0.5,
                "dtype": rng.choice(["bf16", "fp16"]), "page": rng.choice([16, 24, 64]),
                "far": _log(rng, 100, 1000000)}
    if op == "tree":
        B, T, NKV = _log(rng, 1, 32), rng.randint(1, 64), rng.randint(1, 8)
        hi = _log(rng, 16, min(32000, 80000 // B))
        return {"op": op, "B": B, "T": T, "NQ": NKV * rng.choice([g for g in (1, 2, 3, 4, 8) if g * NKV <= 32]),
                "NKV": NKV,
                "D": rng.choice([64, 128]), "page": rng.choice([16, 24, 64, 128]), "lo": rng.choice([0, hi // 2]),
                "hi": hi, "dtype": rng.choice(["bf16", "fp16"]), "chain": rng.random() < 0.3}
    return {"op": op, "B": _log(rng, 1, 256), "V": rng.choice([65536, 50001, 32001, 1009, _log(rng, 2, 65536)]),
            "dtype": rng.choice(["bf16", "fp16", "fp32"]), "temp": rng.choice([0.0, 0.3, 0.7, 1.0, 1.5]),
            "k": rng.choice([0, 1, 20, 50, 1000]), "p": rng.choice([1.0, 0.95, 0.9, 0.5]),
            "minp": rng.choice([0.0, 0.05, 0.2])}


def _spread(lo, hi, n):
    """n lengths from lo to hi, evenly: the same for every seed, so that the work of a case is known."""
    return [lo + (hi - lo) * i // max(n - 1, 1) for i in range(n)]


def _tree_T(c):
    """Drafted tokens of each request: ragged, the largest T, none but the first below one."""
    return [max(1, c["T"] - (i % 4) * (c["T"] // 5)) for i in range(c["B"])]


def work(c):
    op = c["op"]
    if op == "slots":
        lens = _spread(c["lo"], c["hi"], c["B"])
        n = c["B"] * c["add"]
        pages = sum(-(-(l + c["add"]) // c["page"]) - -(-l // c["page"]) for l in lens)
        # two calls: lengths in, granted lengths out, offsets; a position and a slot a token; pages moved both ways
        return {"bytes": 2 * c["B"] * 16 + n * 16 + pages * 16, "flops": 2 * n}
    if op == "rope":
        el = c["N"] * (c["NQ"] + 2 * c["NKV"]) * c["D"]
        return {"bytes": 2 * el * 2 + c["N"] * 16, "flops": el * (6 + (4 if c["norm"] else 0))}
    if op == "tree":
        lens, T, G = _spread(c["lo"], c["hi"], c["B"]), _tree_T(c), c["NQ"]
        kv = sum((l + t) * c["NKV"] * c["D"] * 2 * 2 for l, t in zip(lens, T))
        qo = sum(T) * c["NQ"] * c["D"] * 2 * 2
        return {"bytes": kv + qo, "flops": sum(4 * c["D"] * G * t * (l + (t + 1) / 2) for l, t in zip(lens, T))}
    size = 4 if c["dtype"] == "fp32" else 2
    return {"bytes": c["B"] * c["V"] * size + c["B"] * 28, "flops": 4 * c["B"] * c["V"]}


# ---------------------------------------------------------------------------------------------------- inputs
def _pool(seed, pages):
    return torch.from_numpy(np.random.default_rng(seed).permutation(pages).astype(np.int32))


def prepare(c, seed):
    g = torch.Generator(device=_DEV).manual_seed(seed)
    rn = lambda *s: torch.randn(*s, generator=g, device=_DEV)  # noqa: E731
    op, st = c["op"], {"case": c}
    if op == "slots":
        B, page = c["B"], c["page"]
        rng = np.random.default_rng(seed)
        lens = rng.permutation(np.array(_spread(c["lo"], c["hi"], B)))
        used = -(-lens // page)
        width = int(-(-(c["hi"] + c["add"]) // page) + 1)
        ids = rng.permutation(int(used.sum()) + c["spare"]).astype(np.int32)
        table = np.full((B, width), -1, np.int32)
        at = 0
        for b in range(B):
            table[b, :used[b]] = ids[at:at + used[b]]
            at += int(used[b])
        free = np.full(len(ids), -1, np.int32)
        free[:c["spare"]] = ids[at:]
        i32 = lambda a: torch.from_numpy(np.ascontiguousarray(a, np.int32)).to(_DEV)  # noqa: E731
        n = B * c["add"]
        st.update(lens=i32(lens), new=i32(lens + c["add"]), table=i32(table), free=i32(free),
                  n_free=i32(np.array([c["spare"]])), got=torch.zeros(B, dtype=torch.int32, device=_DEV),
                  back=torch.zeros(B, dtype=torch.int32, device=_DEV),
                  cu=torch.zeros(B + 1, dtype=torch.int32, device=_DEV),
                  cu0=torch.zeros(B + 1, dtype=torch.int32, device=_DEV),
                  positions=torch.full((n,), -1, dtype=torch.int64, device=_DEV),
                  slots=torch.full((n,), -1, dtype=torch.int64, device=_DEV))
    elif op == "rope":
        N, NQ, NKV, D, dt = c["N"], c["NQ"], c["NKV"], c["D"], _DT[c["dtype"]]
        pages = -(-N // c["page"]) + 2
        slots = torch.randperm(pages * c["page"], generator=g, device=_DEV)[:N]
        if N > 8:
            slots[::7] = -1  # padding rows of a batch: nothing of theirs goes into the cache
        inv = 1.0 / (1e6 ** (torch.arange(0, c["rot"], 2, device=_DEV, dtype=torch.float64) / c["rot"]))
        st.update(qkv=rn(N, (NQ + 2 * NKV) * D).to(dt), inv_freq=inv.float(), scaling=1.0,
                  qw=(rn(D) * 0.1 + 1).to(dt) if c["norm"] else None, kw=(rn(D) * 0.1 + 1).to(dt) if c["norm"] else None,
                  positions=torch.randint(0, c["far"], (N,), generator=g, device=_DEV), slots=slots,
                  cached=torch.tensor([n for n in range(N) if N <= 8 or n % 7], device=_DEV),  # rows with a slot
                  q=torch.zeros(N, NQ, D, dtype=dt, device=_DEV), kc=rn(pages, NKV, c["page"], D).to(dt),
                  vc=rn(pages, NKV, c["page"], D).to(dt), eps=1e-5)
    elif op == "tree":
        B, NQ, NKV, D, page, dt = c["B"], c["NQ"], c["NKV"], c["D"], c["page"], _DT[c["dtype"]]
        rng = np.random.default_rng(seed)
        order = rng.permutation(B)  # which request has which length
        ctx, T = [[a[i] for i in order] for a in (_spread(c["lo"], c["hi"], B), _tree_T(c))]
        used = [-(-(l + t) // page) for l, t in zip(ctx, T)]
        pages = sum(used) + 3
        ids = rng.permutation(pages).astype(np.int32)
        table = np.full((B, max(used)), -1, np.int32)
        at, masks = 0, []
        for b in range(B):
            table[b, :used[b]] = ids[at:at + used[b]]
            at += used[b]
            m = []
            for i in range(T[b]):  # an ancestor mask: a node sees itself and its parent's ancestors
                up = 0 if i == 0 else m[i - 1 if c["chain"] else int(rng.integers(max(0, i - 5), i))]
                m.append(up | (1 << i))
            masks += [x - (1 << 64) if x >> 63 else x for x in m]
        N = sum(T)
        cu = np.concatenate([[0], np.cumsum(T)]).astype(np.int32)
        st.update(q=rn(N, NQ, D).to(dt), kc=rn(pages, NKV, page, D).to(dt), vc=rn(pages, NKV, page, D).to(dt),
                  table=torch.from_numpy(table).to(_DEV), ctx=torch.tensor(ctx, dtype=torch.int32, device=_DEV),
                  cu=torch.from_numpy(cu).to(_DEV),
                  mask=None if c["chain"] else torch.tensor(masks, dtype=torch.int64, device=_DEV),
                  out=torch.zeros(N, NQ, D, dtype=dt, device=_DEV), scale=D ** -0.5, ctx_l=ctx, T_l=T, masks_l=masks,
                  host_cu=cu.tolist())
        if own:
            K = _ext()
            S = K.tree_attention_splits(B, NQ, NKV, D, max(T), max(l + t for l, t in zip(ctx, T)))
            st["ws"] = torch.empty(N, NQ, S, D + 2, device=_DEV) if S > 1 else None
    else:
        B, V = c["B"], c["V"]
        x = 2.5 * rn(B, V)
        hot = torch.randint(0, V, (B, 24), generator=g, device=_DEV)  # a few likely continuations a row
        x.scatter_add_(1, hot, 3.0 + 2.0 * rn(B, 24).abs())
        f = lambda v: torch.full((B,), float(v), device=_DEV)  # noqa: E731
        st.update(logits=x.to(_DT[c["dtype"]]), temperature=f(c["temp"]),
                  top_k=torch.full((B,), c["k"], dtype=torch.int32, device=_DEV), top_p=f(c["p"]), min_p=f(c["minp"]),
                  u=torch.rand(B, generator=g, device=_DEV), tok=torch.zeros(B, dtype=torch.int64, device=_DEV))
    return st


# ---------------------------------------------------------------------------------------------------- plain forms
def _plain_slots(lens, new, table, free, n_free, page, got, cu, positions, slots):
    B, width = table.shape
    cap = width * page
    ok = (lens >= 0) & (new >= 0) & (lens <= cap) & (new <= cap)
    old_p, new_p = (lens + page - 1) // page, (new + page - 1) // page
    zero = torch.zeros_like(lens)
    need = torch.where(ok, (new_p - old_p).clamp(min=0), zero)
    tok = torch.where(ok, (new - lens).clamp(min=0), zero)
    ok &= ((need == 0) | (need.cumsum(0) <= n_free)) & ((tok == 0) | (tok.cumsum(0) <= slots.numel()))
    need, tok = torch.where(ok, need, zero), torch.where(ok, tok, zero)
    ret = torch.where(ok, (old_p - new_p).clamp(min=0), zero)
    got.copy_(torch.where(ok, new, lens))
    cu[0] = 0
    cu[1:] = tok.cumsum(0)
    P, R = need.sum(), ret.sum()
    j = torch.arange(width, device=table.device)
    grown = (j >= old_p[:, None]) & (j < (old_p + need)[:, None])
    freed = (j >= (old_p - ret)[:, None]) & (j < old_p[:, None])
    n0 = n_free[0].clone()
    i = (need.cumsum(0) - need)[:, None] + j - old_p[:, None]
    taken = free[(n0 - 1 - i).clamp(0, free.numel() - 1).long()]
    i = (ret.cumsum(0) - ret)[:, None] + j - (old_p - ret)[:, None]
    where = torch.where(freed, n0 - P + R - 1 - i, free.numel()).long()  # the entry past the end takes the rest
    free.copy_(torch.cat([free, free[:1]]).scatter(0, where.flatten(), table.flatten())[:-1])
    table.copy_(torch.where(grown, taken, torch.where(freed, -1, table)))
    n_free.copy_((n_free - P + R))
    t = torch.arange(slots.numel(), device=table.device)
    live = t < cu[-1]
    b = torch.searchsorted(cu[1:], t.int(), right=True).clamp(max=B - 1)
    pos = lens[b].long() + t - cu[b]
    page_id = table[b, (pos // page).clamp(0, width - 1)].long()
    positions.copy_(torch.where(live, pos, positions))
    slots.copy_(torch.where(live, page_id * page + pos % page, slots))


def _plain_rope(st):
    c = st["case"]
    N, NQ, NKV, D, R, page = c["N"], c["NQ"], c["NKV"], c["D"], c["rot"], c["page"]
    x = st["qkv"].view(N, NQ + 2 * NKV, D)
    a = st["positions"].double()[:, None] * st["inv_freq"].double()  # far angles lose their fraction in 32 bits
    cos, sin = (a.cos() * st["scaling"]).float()[:, None], (a.sin() * st["scaling"]).float()[:, None]

    def turn(h, w):
        h = h.float()
        if w is not None:
            h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + st["eps"]) * w.float()
        lo, hi = (h[..., 0:R:2], h[..., 1:R:2]) if c["interleaved"] else (h[..., :R // 2], h[..., R // 2:R])
        a, b = lo * cos - hi * sin, hi * cos + lo * sin
        r = torch.stack([a, b], -1).flatten(-2) if c["interleaved"] else torch.cat([a, b], -1)
        return torch.cat([r, h[..., R:]], -1).to(x.dtype)

    st["q"].copy_(turn(x[:, :NQ], st["qw"]))
    s = st["slots"][st["cached"]]
    st["kc"][s // page, :, s % page] = turn(x[:, NQ:NQ + NKV], st["kw"])[st["cached"]]
    st["vc"][s // page, :, s % page] = x[:, NQ + NKV:][st["cached"]]


def _plain_tree(st):
    c = st["case"]
    NQ, NKV, D = c["NQ"], c["NKV"], c["D"]
    G = NQ // NKV
    for b, (l, t) in enumerate(zip(st["ctx_l"], st["T_l"])):
        n0, L = st["host_cu"][b], l + t
        pages = st["table"][b, :-(-L // c["page"])].long()
        k, v = [x[pages].transpose(0, 1).reshape(NKV, -1, D)[:, :L].float() for x in (st["kc"], st["vc"])]
        q = st["q"][n0:n0 + t].float().view(t, NKV, G, D).permute(1, 0, 2, 3).reshape(NKV, t * G, D)
        s = (q @ k.transpose(1, 2)) * st["scale"]
        j = torch.arange(t, device=q.device)
        if st["mask"] is None:
            see = j[None] <= j[:, None]
        else:
            see = (st["mask"][n0:n0 + t, None] >> j) & 1 != 0
        see = torch.cat([torch.ones(t, l, dtype=torch.bool, device=q.device), see], 1).repeat_interleave(G, 0)
        s.masked_fill_(~see, float("-inf"))
        m = s.amax(-1, keepdim=True)
        p = torch.exp(s - torch.where(m == float("-inf"), torch.zeros_like(m), m))
        z = p.sum(-1, keepdim=True)
        o = (p @ v) / torch.where(z == 0, torch.ones_like(z), z)
        st["out"][n0:n0 + t] = o.view(NKV, t, G, D).permute(1, 0, 2, 3).reshape(t, NQ, D).to(st["out"].dtype)


def _plain_sample(st):
    x = st["logits"].double()  # 64 bits: a running mass next to a border decides a whole number
    B, V = x.shape
    greedy = torch.argmax(st["logits"].float(), -1)
    T = st["temperature"].double()[:, None]
    xs, idx = torch.sort(x, stable=True, dim=-1, descending=True)
    d = xs - xs[:, :1]
    w = torch.exp(d / torch.where(T > 0, T, torch.ones_like(T)))
    rank = torch.arange(V, device=x.device)[None]
    k = st["top_k"].long()[:, None]
    w = torch.where((rank < k) | (k <= 0), w, torch.zeros_like(w))
    p = st["top_p"].double()[:, None]
    run = w.cumsum(-1)
    keep = (run - w < p * run[:, -1:]) | (p >= 1) | (rank == 0)
    keep &= (w >= st["min_p"].double()[:, None].clamp(max=1)) & (w > 0)
    w = torch.zeros_like(w).scatter_(1, idx, torch.where(keep, w, torch.zeros_like(w)))  # back to index order
    run = w.cumsum(-1)
    hit = (run > st["u"].double()[:, None] * run[:, -1:]) & (w > 0)
    st["tok"].copy_(torch.where(T[:, 0] > 0, hit.int().argmax(-1), greedy))


# ---------------------------------------------------------------------------------------------------- one pass
def run(st):
    c, op = st["case"], st["case"]["op"]
    if op == "slots":
        # a round of drafting: pages and slots for the new tokens, and the same pages back when all are turned down
        f = _ext().kv_slots if own else _plain_slots
        f(st["lens"], st["new"], st["table"], st["free"], st["n_free"], c["page"], st["got"], st["cu"],
          st["positions"], st["slots"])
        f(st["got"], st["lens"], st["table"], st["free"], st["n_free"], c["page"], st["back"], st["cu0"],
          st["positions"], st["slots"])
        return {k: st[k] for k in ("got", "cu", "positions", "slots", "back", "cu0", "table", "free", "n_free")}
    if op == "rope":
        if own:
            _ext().qk_norm_rope_kv_paged(st["qkv"], st["qw"], st["kw"], st["inv_freq"], st["scaling"],
                                         st["positions"], st["slots"], st["q"], st["kc"], st["vc"], st["eps"],
                                         c["interleaved"])
        else:
            _plain_rope(st)
        return {k: st[k] for k in ("q", "kc", "vc")}
    if op == "tree":
        if own:
            _ext().tree_attention(st["q"], st["kc"], st["vc"], st["table"], st["ctx"], st["cu"], st["mask"], st["out"],
                                  st["ws"], st["scale"], max(st["T_l"]))
        else:
            _plain_tree(st)
        return st["out"]
    if own:
        _ext().sample_next(st["logits"], st["temperature"], st["top_k"], st["top_p"], st["min_p"], st["u"], st["tok"])
    else:
        _plain_sample(st)
    return st["tok"]


# ---------------------------------------------------------------------------------------------------- 64 bits
def _exact_slots(st):
    c, page = st["case"], st["case"]["page"]
    n = {k: v.cpu().numpy().astype(np.int64) for k, v in st.items() if torch.is_tensor(v)}
    stack = n["free"].copy()

    def turn(lens, new, top, write):
        got, taken, given, offs, total_need, total_tok = [], [], [], [0], 0, 0
        width = n["table"].shape[1]
        for b in range(c["B"]):
            l, w = int(lens[b]), int(new[b])
            fits = 0 <= l <= width * page and 0 <= w <= width * page
            pl, pw = math.ceil(l / page), math.ceil(w / page)
            need, tok = (max(pw - pl, 0), max(w - l, 0)) if fits else (0, 0)
            total_need, total_tok = total_need + need, total_tok + tok
            fits = fits and (not need or total_need <= top) and (not tok or total_tok <= len(n["slots"]))
            got.append(w if fits else l)
            if fits:
                for j in range(pl, pw):
                    n["table"][b, j] = stack[top - 1 - len(taken)]
                    taken.append(j)
                for j in range(pw, pl):
                    given.append((b, j))
                for i, pos in enumerate(range(l, w)):
                    n["positions"][offs[-1] + i] = pos
                    n["slots"][offs[-1] + i] = n["table"][b, pos // page] * page + pos % page
            offs.append(offs[-1] + (tok if fits else 0))
        top = top - len(taken) + len(given)
        for i, (b, j) in enumerate(given):
            stack[top - 1 - i] = n["table"][b, j]
            n["table"][b, j] = -1
        n[write[0]], n[write[1]] = np.array(got), np.array(offs)
        return top

    top = turn(n["lens"], n["new"], int(n["n_free"][0]), ("got", "cu"))
    top = turn(n["got"], n["lens"], top, ("back", "cu0"))
    n["free"], n["n_free"] = stack, np.array([top])
    return {k: torch.from_numpy(n[k]).to(_DEV).to(st[k].dtype)
            for k in ("got", "cu", "positions", "slots", "back", "cu0", "table", "free", "n_free")}


def _exact_rope(st):
    c = st["case"]
    N, NQ, NKV, D, R, page = c["N"], c["NQ"], c["NKV"], c["D"], c["rot"], c["page"]
    x = st["qkv"].double().view(N, NQ + 2 * NKV, D)
    # the pairs as complex numbers, turned by e^(i angle)
    ang = torch.outer(st["positions"].double(), st["inv_freq"].double())
    e = torch.polar(torch.full_like(ang, st["scaling"]), ang)
    i = torch.arange(R // 2, device=x.device)
    first, second = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + R // 2)
    y = x.clone()
    for lo, n, w in ((0, NQ, st["qw"]), (NQ, NKV, st["kw"])):
        h = y[:, lo:lo + n]
        if w is not None:
            h = w.double() * h / torch.sqrt((h * h).sum(-1, keepdim=True) / D + st["eps"])
        z = torch.complex(h[..., first], h[..., second]) * e[:, None]
        h = h.clone()
        h[..., first], h[..., second] = z.real, z.imag
        y[:, lo:lo + n] = h
    kc, vc = st["kc"].double(), st["vc"].double()
    for cache, lo in ((kc, NQ), (vc, NQ + NKV)):
        rows = cache.transpose(1, 2).clone(memory_format=torch.contiguous_format).view(-1, NKV, D)
        keep = st["slots"] >= 0
        rows[st["slots"][keep]] = y[keep, lo:lo + NKV]
        cache.copy_(rows.view(-1, page, NKV, D).transpose(1, 2))
    return {"q": y[:, :NQ].contiguous(), "kc": kc, "vc": vc}


def _exact_tree(st):
    c = st["case"]
    NKV, D, page = c["NKV"], c["D"], c["page"]
    G, out = c["NQ"] // NKV, torch.zeros(st["q"].shape, dtype=torch.float64, device=_DEV)
    for b in range(c["B"]):
        n0, l, t = int(st["cu"][b]), st["ctx_l"][b], st["T_l"][b]
        pos = torch.arange(l + t, device=_DEV)
        pid = st["table"][b].long()[pos // page]
        see = np.ones((t, l + t), bool)
        for i in range(t):
            for j in range(t):
                see[i, l + j] = (st["masks_l"][n0 + i] >> j) & 1
        see = torch.from_numpy(see).to(_DEV)
        for h in range(NKV):
            k, v = st["kc"][pid, h, pos % page].double(), st["vc"][pid, h, pos % page].double()
            for gq in range(G):
                s = st["scale"] * (st["q"][n0:n0 + t, h * G + gq].double() @ k.T)
                p = torch.softmax(s.masked_fill(~see, float("-inf")), -1)
                out[n0:n0 + t, h * G + gq] = torch.where(see.any(-1, keepdim=True), p @ v, torch.zeros_like(p @ v))
    return out


def _exact_sample(st):
    c, toks = st["case"], []
    T, k, p, mp, u = [st[n].double().cpu().numpy() for n in ("temperature", "top_k", "top_p", "min_p", "u")]
    for b, row in enumerate(st["logits"].double().cpu().numpy()):
        if not T[b] > 0:
            toks.append(int(np.argmax(row)))
            continue
        order = np.argsort(-row, kind="stable")
        if k[b] > 0:
            order = order[:int(k[b])]
        w = np.exp((row[order] - row[order[0]]) / T[b])
        if p[b] < 1:
            order = order[:1 + int(np.searchsorted(np.cumsum(w), p[b] * w.sum()))]
        w = w[:len(order)]
        order = np.sort(order[(w >= min(mp[b], 1.0)) & (w > 0)])
        cum = np.cumsum(np.exp((row[order] - row.max()) / T[b]))
        toks.append(int(order[np.searchsorted(cum, u[b] * cum[-1], side="right")]))
    return torch.tensor(toks, dtype=torch.int64, device=_DEV)


def exact(c, seed):
    st = prepare(c, seed)
    return {"slots": _exact_slots, "rope": _exact_rope, "tree": _exact_tree, "sample": _exact_sample}[c["op"]](st)
