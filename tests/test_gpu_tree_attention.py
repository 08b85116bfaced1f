"""Attention of drafted tokens over a paged cache (tree_attention) on the B200, against 64 bits.

Tolerance, from the arithmetic: every probability is rounded once to the type (eps / 2 of it) before the second product
while the sum keeps it unrounded, the output once more; fp32 sums and exponentials of up to some thousand terms add less
than 2e-5 of the largest |v|. So |err| <= eps / 2 (|out| + sum_t p_t |v_t|) + 2e-5 max |v|, and sum p |v| <= max |v|:
the bound used is eps / 2 (|out| + max |v|) + 2e-5 max |v|, max |v| over the request's values of that head.
"""

import numpy as np
import pytest
import torch

from lfm2opt.kernels import ext
from oracle.serving import tree_attention_f64

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


def make(seed, NQ, NKV, D, page, ctx, T, dt, chain=False, spare=2, pad_rows=0, width=None):
    """CPU tensors of a batch: random trees (masks as Python ints), pages in random order."""
    rng = np.random.default_rng(seed)
    g = torch.Generator().manual_seed(seed)
    used = [-(-(c + t) // page) for c, t in zip(ctx, T)]
    pages = sum(used) + spare
    ids = rng.permutation(pages)
    table = np.full((len(ctx), width or max(max(used), 1)), -1, np.int32)
    at, masks = 0, []
    for b, n in enumerate(used):
        table[b, :n] = ids[at:at + n]
        at += n
        m = []
        for i in range(T[b]):
            up = 0 if i == 0 else m[i - 1 if chain else int(rng.integers(max(0, i - 4), i))]
            m.append(up | (1 << i))
        masks += m
    N = sum(T) + pad_rows
    masks += [0] * pad_rows
    cu = np.concatenate([[0], np.cumsum(T)]).astype(np.int32)
    rn = lambda *s: torch.randn(*s, generator=g).to(DT[dt])  # noqa: E731
    return dict(q=rn(N, NQ, D), kc=rn(pages, NKV, page, D), vc=rn(pages, NKV, page, D),
                table=torch.from_numpy(table), ctx=torch.tensor(ctx, dtype=torch.int32), cu=torch.from_numpy(cu),
                mask=None if chain else masks, scale=D ** -0.5, max_q=max(max(T), 1))


def signed(masks):
    return torch.tensor([m - (1 << 64) if m >> 63 else m for m in masks], dtype=torch.int64)


def run(dev, c, S=None):
    N, NQ, D = c["q"].shape
    d = {k: v.to(dev) for k, v in c.items() if torch.is_tensor(v)}
    out = torch.full(c["q"].shape, float("nan"), dtype=c["q"].dtype, device=dev)
    if S is None:
        S = ext().tree_attention_splits(len(c["ctx"]), NQ, c["kc"].shape[1], D, c["max_q"],
                                        c["table"].shape[1] * c["kc"].shape[2])
    ws = torch.full((N, NQ, S, D + 2), float("nan"), device=dev) if S > 1 else None
    ext().tree_attention(d["q"], d["kc"], d["vc"], d["table"], d["ctx"], d["cu"],
                         None if c["mask"] is None else signed(c["mask"]).to(dev), out, ws, c["scale"], c["max_q"])
    torch.cuda.synchronize()
    return out


def reference(c):
    return tree_attention_f64(c["q"], c["kc"], c["vc"], c["table"], c["ctx"], c["cu"], c["mask"], c["scale"],
                              c["max_q"])


def check(out, ref, c):
    vmax = c["vc"].float()
    vmax = vmax[vmax.isfinite()].abs().max().item()
    out = out.cpu().double()
    assert torch.equal(out.isnan(), ref.isnan())  # rows outside the requests: as they were
    err, lim = (out - ref).abs(), torch.finfo(c["q"].dtype).eps / 2 * (ref.abs() + vmax) + 2e-5 * vmax
    ok = ref.isnan() | (err <= lim)
    assert ok.all(), (err[~ok].max().item(), (~ok).nonzero()[:4].tolist())


CASES = [
    # NQ, NKV, D, page, ctx, T, dt, chain
    (32, 8, 64, 64, [1000], [1], "bf16", True),
    (4, 1, 64, 16, [0], [1], "fp16", True),
    (8, 8, 64, 1, [5, 0, 17], [1, 2, 3], "bf16", False),
    (32, 8, 64, 64, [0, 63, 64, 200], [8, 8, 7, 1], "bf16", False),
    (24, 3, 128, 16, [0, 100, 777], [13, 2, 4], "fp16", False),
    (16, 2, 128, 24, [300, 50], [16, 9], "bf16", False),
    (6, 2, 64, 7, [129, 1], [64, 33], "fp16", False),
    (8, 1, 128, 128, [400], [64], "bf16", True),
    (64, 1, 64, 32, [90], [5], "bf16", False),
    (12, 4, 128, 64, [0, 0], [0, 21], "fp16", False),
]


@pytest.mark.parametrize("S", [None, 1, 3])
@pytest.mark.parametrize("NQ,NKV,D,page,ctx,T,dt,chain", CASES)
def test_tree_attention_against_64_bits(cuda_dev, NQ, NKV, D, page, ctx, T, dt, chain, S):
    c = make(len(ctx) + NQ + page, NQ, NKV, D, page, ctx, T, dt, chain, pad_rows=3)
    check(run(cuda_dev, c, S), reference(c), c)


@pytest.mark.parametrize("max_ctx,B,T", [(2500, 3, 16), (2500, 1, 1), (2000, 2, 64)])
def test_longer_contexts(cuda_dev, max_ctx, B, T):
    c = make(B, 8, 2, 64, 16, [max_ctx - 700 * b for b in range(B)], [T] * B, "bf16")
    check(run(cuda_dev, c), reference(c), c)


def test_queries_that_see_nothing_give_zeros(cuda_dev):
    c = make(1, 8, 2, 64, 16, [0, 0, 40], [5, 1, 3], "bf16")
    c["mask"] = [0, 1, 0, 12, 0, 0, 0, 7, 0]
    out, ref = run(cuda_dev, c), reference(c)
    check(out, ref, c)
    assert torch.count_nonzero(out[[0, 2, 4, 5]]) == 0


def test_masked_infinities_and_nans_do_not_spread(cuda_dev):
    """Drafts that hold an infinity or a NaN reach the queries that see them and no others; stale rows behind the
    length and unused pages are never read into a result."""
    for D, dt, T in ((64, "bf16", 7), (128, "fp16", 20), (64, "fp16", 64)):
        c = make(3, 8, 2, D, 16, [70, 33], [T, 5], dt, spare=2)
        k, v = c["kc"], c["vc"]
        live = torch.zeros(k.shape[0], 16, dtype=torch.bool)
        for b, L in enumerate((70 + T, 38)):
            for t in range(L):
                live[c["table"][b, t // 16], t % 16] = True
        k.transpose(1, 2)[~live] = float("nan")
        v.transpose(1, 2)[~live] = float("inf")
        poison = 70 + 3  # draft 3 of request 0
        pg, r = int(c["table"][0, poison // 16]), poison % 16
        v[pg, 0, r, 5], v[pg, 1, r, D - 1], k[pg, 0, r, 2] = float("inf"), float("nan"), float("nan")
        sees = [bool((m >> 3) & 1) for m in c["mask"][:T]]
        clean = dict(c, kc=k.clone(), vc=v.clone())
        clean["kc"].nan_to_num_(0, 0, 0), clean["vc"].nan_to_num_(0, 0, 0)
        for S in (1, 2):
            out, ref = run(cuda_dev, c, S), reference(clean)
            blind = [i for i in range(T) if not sees[i]] + list(range(T, T + 5))
            check(out[blind], ref[blind], clean)
            seeing = [i for i in range(T) if sees[i]]
            assert not out[seeing, :4].isfinite().all(-1).any() and out[seeing, 4:, D - 1].isnan().all()


def test_pages_outside_the_pool_are_not_seen(cuda_dev):
    c = make(4, 8, 2, 64, 16, [100, 30], [4, 4], "bf16")
    c["table"][0, 2], c["table"][1, 0] = -1, c["kc"].shape[0]
    check(run(cuda_dev, c, 2), reference(c), c)
    c["ctx"][1] = 100000  # past the table: what the table holds
    check(run(cuda_dev, c), reference(c), c)


def test_more_queries_than_max_q_are_left(cuda_dev):
    c = make(5, 4, 1, 64, 16, [20], [9], "bf16")
    c["max_q"] = 6
    out = run(cuda_dev, c)
    assert out[6:].isnan().all()
    ref = tree_attention_f64(c["q"], c["kc"], c["vc"], c["table"], c["ctx"], c["cu"], c["mask"], c["scale"], 6)
    check(out, ref, c)


def test_dense_cache_is_one_page_per_request(cuda_dev):
    """page = max_len and table[b] = {b}: the cache of decode_attention_split, and its result."""
    g = torch.Generator().manual_seed(9)
    B, NKV, L, pos = 3, 8, 777, 500
    q = torch.randn(B, 32, 64, generator=g).bfloat16().to(cuda_dev)
    kc, vc = [torch.randn(B, NKV, L, 64, generator=g).bfloat16().to(cuda_dev) for _ in range(2)]
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda_dev)  # noqa: E731
    a, b = torch.empty_like(q), torch.empty_like(q)
    ext().decode_attention_split(q, kc, vc, torch.tensor([pos], device=cuda_dev), a,
                                 torch.empty(B, 32, 4, 66, device=cuda_dev), 0.125)
    ext().tree_attention(q, kc, vc, i32([[0], [1], [2]]), i32([pos] * B), i32([0, 1, 2, 3]), None, b, None, 0.125, 1)
    # two roundings of the output and one of every probability
    lim = torch.finfo(q.dtype).eps / 2 * (2 * a.float().abs() + vc.float().abs().max()) + 4e-5 * vc.float().abs().max()
    assert ((a.float() - b.float()).abs() <= lim).all()


def test_repeatable_and_capturable(cuda_dev):
    c = make(6, 32, 8, 64, 64, [900, 64], [16, 3], "bf16")
    first = run(cuda_dev, c)
    assert torch.equal(first.nan_to_num(), run(cuda_dev, c).nan_to_num())
    d = {k: v.to(cuda_dev) for k, v in c.items() if torch.is_tensor(v)}
    mask, out = signed(c["mask"]).to(cuda_dev), torch.full_like(first, float("nan"))
    S = ext().tree_attention_splits(2, 32, 8, 64, 16, 1024)
    ws = torch.empty(19, 32, S, 66, device=cuda_dev) if S > 1 else None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ext().tree_attention(d["q"], d["kc"], d["vc"], d["table"], d["ctx"], d["cu"], mask, out, ws, c["scale"], 16)
    d["q"].zero_()
    graph.replay()  # uniform attention over what is seen
    torch.cuda.synchronize()
    zero = dict(c, q=torch.zeros_like(c["q"]))
    check(out, reference(zero), zero)


def test_long_cache_offsets_pass_32_bits(cuda_dev):
    """A pool whose last page starts behind 2^32 elements: the request sits at its far end."""
    NKV, page, D = 8, 64, 64
    pages = (1 << 32) // (NKV * page * D) + 5  # 8.6 GB a cache
    kc = torch.zeros(pages, NKV, page, D, dtype=torch.bfloat16, device=cuda_dev)
    vc = torch.zeros_like(kc)
    c = make(8, 32, NKV, D, page, [150], [3], "bf16", spare=0)
    ids = torch.tensor([pages - 1, 0, pages - 3])
    kc[ids.to(cuda_dev)], vc[ids.to(cuda_dev)] = c["kc"][c["table"][0].long()].to(cuda_dev), \
        c["vc"][c["table"][0].long()].to(cuda_dev)
    q = c["q"].to(cuda_dev)
    out = torch.full_like(q, float("nan"))
    i32 = lambda t: t.to(torch.int32).to(cuda_dev)  # noqa: E731
    ext().tree_attention(q, kc, vc, i32(ids)[None], i32(c["ctx"]), i32(c["cu"]), signed(c["mask"]).to(cuda_dev), out,
                         None, c["scale"], 3)
    check(out, reference(c), c)


def test_refusals(cuda_dev):
    c = make(7, 8, 2, 64, 16, [20], [3], "bf16")
    d = {k: v.to(cuda_dev) for k, v in c.items() if torch.is_tensor(v)}
    out, m = torch.empty_like(d["q"]), signed(c["mask"]).to(cuda_dev)

    def call(**kw):
        a = dict(d, mask=m, out=out, ws=None, scale=0.125, max_q=3, **{})
        a.update(kw)
        ext().tree_attention(a["q"], a["kc"], a["vc"], a["table"], a["ctx"], a["cu"], a["mask"], a["out"], a["ws"],
                             a["scale"], a["max_q"])

    for kw, match in ((dict(max_q=65), "max_q"), (dict(max_q=0), "max_q"), (dict(scale=0.0), "scale"),
                      (dict(q=d["q"].float(), out=out.float()), "bf16 or fp16"), (dict(mask=m[:2]), "mask"),
                      (dict(kc=d["kc"].half()), "dtype"), (dict(cu=d["cu"][:1]), "cu"),
                      (dict(table=d["table"].long()), "int32"), (dict(q=d["q"][:, :3]), "contiguous"),
                      (dict(ws=torch.empty(3, 8, 2, 64, device=cuda_dev)), "ws")):
        with pytest.raises(RuntimeError, match=match):
            call(**kw)


@pytest.mark.parametrize("D,dt,T,S", [(64, "bf16", 3, 1), (64, "fp16", 40, 4), (128, "bf16", 9, 3), (128, "fp16", 64, 2),
                                      (64, "bf16", 64, 1)])
@pytest.mark.parametrize("order", ["growing", "falling", "jumping"])
def test_maxima_that_move_along_the_cache(cuda_dev, D, dt, T, S, order):
    """Scores whose maximum grows by more than 2^8 from tile to tile (the accumulator is rescaled in every one, the last
    included), falls, or jumps."""
    c = make(11, 8, 2, D, 16, [450, 130], [T, 2], dt)
    direction = torch.randn(D, generator=torch.Generator().manual_seed(5))
    direction /= direction.norm()
    for b in range(2):
        L = int(c["ctx"][b]) + (T if b == 0 else 2)
        for t in range(L):
            step = t // 16 if order == "growing" else -(t // 16) if order == "falling" else (t // 64) * 37 % 29
            k = c["kc"][int(c["table"][b, t // 16]), :, t % 16]
            k.copy_((0.2 * k.float() + 4.0 * step * direction).to(k.dtype))
    c["q"] = (0.3 * c["q"].float() + 4.0 * direction).to(c["q"].dtype)
    check(run(cuda_dev, c, S), reference(c), c)


def test_more_parts_than_a_warp_has_lanes(cuda_dev):
    c = make(12, 8, 2, 64, 64, [4500], [2], "bf16")  # 71 tiles
    for S in (70, 40):
        check(run(cuda_dev, c, S), reference(c), c)


@pytest.mark.parametrize("page", [8, 24, 40, 5, 200])
def test_page_sizes_that_tiles_straddle(cuda_dev, page):
    for D, T in ((64, 6), (128, 40)):
        c = make(page, 12, 3, D, page, [333, 64], [T, T], "fp16")
        check(run(cuda_dev, c, 3), reference(c), c)


def test_many_requests_with_and_without_queries(cuda_dev):
    """More requests than a warp has lanes and blocks have stretches; some bring nothing."""
    rng = np.random.default_rng(13)
    ctx, T = rng.integers(0, 150, 300).tolist(), rng.integers(0, 4, 300).tolist()
    c = make(13, 4, 2, 64, 16, ctx, T, "bf16")
    for S in (1, 3):
        check(run(cuda_dev, c, S), reference(c), c)


def test_two_streams_at_once(cuda_dev):
    """Calls with workspaces of their own on two streams, among other kernels that use tensor memory."""
    from lfm2opt.kernels import check_device, int8_ext
    cs = [make(20 + i, 32, 8, 64, 64, [700, 300], [16, 9], "bf16") for i in range(2)]
    refs = [reference(c) for c in cs]
    streams = [torch.cuda.Stream(cuda_dev) for _ in cs]
    xq = torch.randint(-127, 128, (512, 1024), dtype=torch.int8, device=cuda_dev)
    sx, y = torch.ones(512, device=cuda_dev), torch.empty(512, 512, dtype=torch.bfloat16, device=cuda_dev)
    work = []
    for c in cs:
        d = {k: v.to(cuda_dev) for k, v in c.items() if torch.is_tensor(v)}
        work.append((d, signed(c["mask"]).to(cuda_dev), torch.full_like(d["q"], float("nan")),
                     torch.empty(25, 32, 6, 66, device=cuda_dev)))
    torch.cuda.synchronize()
    for _ in range(10):
        for s, c, (d, m, out, ws) in zip(streams, cs, work):
            with torch.cuda.stream(s):
                ext().tree_attention(d["q"], d["kc"], d["vc"], d["table"], d["ctx"], d["cu"], m, out, ws, c["scale"], 16)
        with torch.cuda.stream(streams[0]):
            int8_ext().gemm_i8(xq, sx, xq, sx, None, y, False)
    torch.cuda.synchronize()
    for c, ref, (_, _, out, _) in zip(cs, refs, work):
        check(out, ref, c)
    check_device()


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("NQ,T", [(8, 1), (8, 3), (32, 16), (32, 64)])
def test_long_units_of_wide_heads(cuda_dev, NQ, T, dt):
    """Heads of 128: more tiles than stages in one block, one row tile and two, units cut in parts of many lengths."""
    c = make(40 + T, NQ, NQ // 4, 128, 32, [3000, 70], [T, T], dt)
    for S in (None, 1, 2, 9):
        check(run(cuda_dev, c, S), reference(c), c)


@pytest.mark.parametrize("D", [64, 128])
def test_many_units_in_a_block(cuda_dev, D):
    """More units than blocks have stretches: several units, whole and cut ones, follow each other in a block."""
    rng = np.random.default_rng(D)
    ctx, T = rng.integers(0, 400, 260).tolist(), rng.integers(1, 3, 260).tolist()
    c = make(14, 16, 4, D, 64, ctx, T, "bf16")
    for S in (1, 2, 4):
        check(run(cuda_dev, c, S), reference(c), c)


def test_other_workspaces_contents_do_not_matter(cuda_dev):
    """The joining kernel reads what this call's parts wrote: the same bits over any contents of the workspace."""
    c = make(15, 32, 8, 64, 64, [1500, 200, 40], [5, 16, 1], "bf16")
    d = {k: v.to(cuda_dev) for k, v in c.items() if torch.is_tensor(v)}
    outs = []
    for fill in (0.0, 1e30, float("inf"), -1.0):
        out, ws = torch.zeros_like(d["q"]), torch.full((22, 32, 20, 66), fill, device=cuda_dev)
        ext().tree_attention(d["q"], d["kc"], d["vc"], d["table"], d["ctx"], d["cu"], signed(c["mask"]).to(cuda_dev), out,
                             ws, c["scale"], 16)
        outs.append(out.cpu())
    check(outs[0], reference(c), c)
    assert all(torch.equal(outs[0], o) for o in outs[1:])


@pytest.mark.parametrize("page", [64, 20])
@pytest.mark.parametrize("D,T,n,drop", [(64, 1, 32000, 17.34375), (128, 3, 32000, 17.34375), (64, 40, 131072, 17.34375),
                                        (64, 1, 131072, 21.0), (128, 40, 40000, 19.5)])
def test_many_small_probabilities_in_fp16(cuda_dev, D, T, n, drop, page):
    """One key above many whose probabilities, e^-drop, lie below fp16's smallest step: together they still count. All
    in one part, so that the one key's maximum holds for every other."""
    c = make(50, 2, 1, D, page, [n], [T], "fp16", chain=True)
    c["q"].zero_(), c["kc"].zero_(), c["vc"].fill_(1.0)
    c["q"][:, :, 0] = 8.0
    c["scale"] = 0.125
    pg, r = int(c["table"][0, 777 // page]), 777 % page
    c["kc"][pg, 0, r, 0], c["vc"][pg, 0, r] = drop, 0.0
    check(run(cuda_dev, c, 1), reference(c), c)


# ----------------------------------------------------------------------------- pages that are not multiples of 8
@pytest.mark.parametrize("S", [1, 3])
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("NQ,NKV,T", [(4, 2, 1), (8, 2, 4), (24, 3, 3), (8, 2, 8), (12, 3, 16), (10, 1, 7), (16, 2, 40)])
def test_other_pages_every_block_shape(cuda_dev, NQ, NKV, T, D, S):
    """2, 16, 24, 32, 64, 70 and 320 rows a KV head: every split of warps over rows and keys, odd numbers of rows."""
    c = make(60 + T, NQ, NKV, D, 20, [500, 61, 0], [T, max(1, T - 1), 1], ("bf16", "fp16")[T % 2])
    check(run(cuda_dev, c, S), reference(c), c)


@pytest.mark.parametrize("D", [64, 128])
def test_other_pages_queries_that_see_nothing(cuda_dev, D):
    c = make(1, 8, 2, D, 20, [0, 0, 40], [5, 1, 3], "bf16")
    c["mask"] = [0, 1, 0, 12, 0, 0, 0, 7, 0]
    for S in (1, 2):
        out = run(cuda_dev, c, S)
        check(out, reference(c), c)
        assert torch.count_nonzero(out[[0, 2, 4, 5]]) == 0


@pytest.mark.parametrize("page", [20, 7])
@pytest.mark.parametrize("D,dt,T", [(64, "bf16", 4), (64, "fp16", 7), (64, "bf16", 14), (64, "fp16", 64), (128, "bf16", 4),
                                    (128, "fp16", 6), (128, "bf16", 16), (128, "fp16", 20)])
def test_other_pages_masked_infinities_and_nans(cuda_dev, D, dt, T, page):
    c = make(3, 8, 2, D, page, [70, 33], [T, 3], dt, spare=2)
    k, v = c["kc"], c["vc"]
    live = torch.zeros(k.shape[0], page, dtype=torch.bool)
    for b, L in enumerate((70 + T, 36)):
        for t in range(L):
            live[c["table"][b, t // page], t % page] = True
    k.transpose(1, 2)[~live] = float("nan")
    v.transpose(1, 2)[~live] = float("inf")
    poison = 70 + 2  # draft 2 of request 0
    pg, r = int(c["table"][0, poison // page]), poison % page
    v[pg, 0, r, 5], v[pg, 1, r, D - 1], k[pg, 0, r, 2] = float("inf"), float("nan"), float("nan")
    sees = [bool((m >> 2) & 1) for m in c["mask"][:T]]
    clean = dict(c, kc=k.clone(), vc=v.clone())
    clean["kc"].nan_to_num_(0, 0, 0), clean["vc"].nan_to_num_(0, 0, 0)
    for S in (1, 2):
        out, ref = run(cuda_dev, c, S), reference(clean)
        blind = [i for i in range(T) if not sees[i]] + list(range(T, T + 3))
        check(out[blind], ref[blind], clean)
        seeing = [i for i in range(T) if sees[i]]
        assert not out[seeing, :4].isfinite().all(-1).any() and out[seeing, 4:, D - 1].isnan().all()


@pytest.mark.parametrize("D", [64, 128])
def test_other_pages_outside_the_pool_and_past_max_q(cuda_dev, D):
    c = make(4, 8, 2, D, 20, [100, 30], [4, 4], "bf16")
    c["table"][0, 2], c["table"][1, 0] = -1, c["kc"].shape[0]
    for S in (1, 2):
        check(run(cuda_dev, c, S), reference(c), c)
    c["ctx"][1] = 100000  # past the table: what the table holds
    check(run(cuda_dev, c), reference(c), c)
    c = make(5, 4, 1, D, 20, [20], [9], "bf16")
    c["max_q"] = 6
    out = run(cuda_dev, c)
    assert out[6:].isnan().all()
    check(out, tree_attention_f64(c["q"], c["kc"], c["vc"], c["table"], c["ctx"], c["cu"], c["mask"], c["scale"], 6), c)


@pytest.mark.parametrize("D,dt,T,S", [(64, "bf16", 3, 1), (64, "fp16", 7, 3), (64, "bf16", 40, 2), (128, "fp16", 4, 3),
                                      (128, "bf16", 8, 1), (128, "fp16", 16, 2), (128, "bf16", 64, 1)])
@pytest.mark.parametrize("order", ["growing", "falling", "jumping"])
def test_other_pages_maxima_that_move(cuda_dev, D, dt, T, S, order):
    c = make(11, 8, 2, D, 20, [450, 130], [T, 2], dt)
    direction = torch.randn(D, generator=torch.Generator().manual_seed(5))
    direction /= direction.norm()
    for b in range(2):
        L = int(c["ctx"][b]) + (T if b == 0 else 2)
        for t in range(L):
            step = t // 16 if order == "growing" else -(t // 16) if order == "falling" else (t // 64) * 37 % 29
            k = c["kc"][int(c["table"][b, t // 20]), :, t % 20]
            k.copy_((0.2 * k.float() + 4.0 * step * direction).to(k.dtype))
    c["q"] = (0.3 * c["q"].float() + 4.0 * direction).to(c["q"].dtype)
    check(run(cuda_dev, c, S), reference(c), c)
