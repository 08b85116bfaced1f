"""Sampling (sample_next) on the B200: whole numbers, equal to the definition in 64 bits.

The kernel sums weights in steps of 2^-44 of the largest; on the fixed seeds here no draw falls within that of a border,
so every token is equal.
"""

import numpy as np
import pytest
import torch

from lfm2opt.kernels import ext
from oracle.serving import sample_next_f64

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def draw(dev, x, temperature=None, top_k=None, top_p=None, min_p=None, u=None, pos=None):
    B = x.shape[0]
    f = lambda a, t=torch.float32: None if a is None else torch.tensor(a, dtype=t, device=dev)  # noqa: E731
    tok = torch.full((B,), -1, dtype=torch.int64, device=dev)
    ext().sample_next(x.to(dev) if not x.is_cuda else x, f(temperature), f(top_k, torch.int32), f(top_p), f(min_p),
                      f(u), tok, pos)
    return tok.cpu().tolist()


def want(x, temperature, top_k, top_p, min_p, u):
    r = np.float32  # the kernel takes fp32 parameters
    return [sample_next_f64(row.double().numpy(), float(r(t)), k, float(r(p)), float(r(m)), float(r(v)))
            for row, t, k, p, m, v in zip(x.cpu(), temperature, top_k, top_p, min_p, u)]


def params(rng, B):
    pick = lambda *a: [a[i] for i in rng.integers(0, len(a), B)]  # noqa: E731
    return dict(temperature=pick(0.0, 0.2, 0.7, 1.0, 3.0), top_k=pick(0, 0, 1, 2, 40, 1000, 10**6),
                top_p=pick(1.0, 0.95, 0.9, 0.5, 0.01, 0.0), min_p=pick(0.0, 0.0, 0.05, 0.5, 1.0),
                u=rng.random(B, dtype=np.float32).tolist())


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("V", [1, 2, 7, 8, 33, 1009, 4096, 50001, 65536])
def test_equal_to_the_definition(cuda_dev, V, dt):
    rng = np.random.default_rng(V)
    B = 40 if V < 5000 else 16
    g = torch.Generator().manual_seed(V)
    x = (2.5 * torch.randn(B, V, generator=g) + 6 * (torch.rand(B, V, generator=g) < 20 / V)).to(DT[dt])
    p = params(rng, B)
    assert draw(cuda_dev, x, **p) == want(x, **p)


@pytest.mark.parametrize("B", [1, 3, 200])
def test_batch_sizes_and_strided_rows(cuda_dev, B):
    """One row spread over a cluster, and a batch of one block a row; rows 2 bytes off any alignment."""
    g = torch.Generator().manual_seed(B)
    wide = (3 * torch.randn(B, 9003, generator=g)).bfloat16().to(cuda_dev)
    x = wide[:, 1:9002]
    p = params(np.random.default_rng(B), B)
    assert draw(cuda_dev, x, **p) == want(x, **p)


def test_largest_vocabulary(cuda_dev):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 1 << 18, generator=g) * 2
    for dt in DT.values():
        p = dict(temperature=[1.0, 0.9], top_k=[0, 5000], top_p=[0.97, 0.99], min_p=[0.0, 0.0], u=[0.83, 0.4])
        assert draw(cuda_dev, x.to(dt), **p) == want(x.to(dt), **p)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
def test_ties_infinities_and_nans(cuda_dev, dt):
    inf, nan = float("inf"), float("nan")
    V = 3000
    rows, p = [], dict(temperature=[], top_k=[], top_p=[], min_p=[], u=[])

    def add(row, T=1.0, k=0, tp=1.0, mp=0.0, u=0.5):
        rows.append(row)
        for n, v in zip(p, (T, k, tp, mp, u)):
            p[n].append(v)

    flat = torch.zeros(V)
    for u in (0.0, 0.1234, 0.999999):
        add(flat, u=u)                      # all equal
        add(flat, k=7, u=u)                 # ties at the cut: the lowest indexes
        add(flat, tp=0.25, u=u)
        add(flat, k=1000, tp=0.5, u=u)
        add(flat, mp=1.0, u=u)
    some = torch.full((V,), -inf)
    some[[5, 99, 2000]] = torch.tensor([1.0, 2.0, 1.0])
    for u in (0.0, 0.3, 0.99):
        add(some, u=u)
        add(some, k=2, u=u)                 # one of two equal ones: the lower index
        add(some, k=500, tp=0.999, u=u)     # more asked for than there is mass
    add(torch.full((V,), -inf))             # nothing finite: the first
    top = flat.clone()
    top[[17, 30]] = inf
    add(top, u=0.2), add(top, u=0.7), add(top, k=1), add(top, T=0.0)
    bad = flat.clone()
    bad[40], bad[41] = nan, nan
    add(bad), add(bad, T=0.0)
    signs = torch.where(torch.arange(V) % 2 == 0, -0.0, 0.0)
    add(signs, k=3, u=0.9), add(signs, k=3, u=0.1)  # zeros of both signs are one value
    tiny = torch.zeros(V)
    tiny[:4] = torch.tensor([1e-30, -1e-30, 2e-38, -2e-38])
    add(tiny, k=2, u=0.9), add(tiny, k=4, u=0.9), add(tiny, tp=0.001, u=0.9)
    spread = torch.linspace(-60000, 60000, V)
    add(spread, T=1e-3, u=0.5), add(spread, T=1e6, tp=0.5, u=0.5), add(spread, T=1e30, u=0.7), add(spread, T=inf, u=0.7)
    add(spread, T=nan), add(spread, tp=nan, T=30.0), add(spread, mp=nan, T=30.0), add(spread, T=-1.0)
    add(spread, T=30.0, mp=7.0, u=0.9), add(spread, T=30.0, tp=-1.0, u=0.9), add(spread, T=30.0, k=-4, u=0.9)
    x = torch.stack(rows).to(DT[dt])
    assert draw(cuda_dev, x, **p) == want(x, **p)


def test_off_switches_and_position(cuda_dev):
    g = torch.Generator().manual_seed(1)
    x = torch.randn(4, 500, generator=g)
    u = [0.1, 0.4, 0.6, 0.9]
    pos = torch.tensor([41], device=cuda_dev)
    assert draw(cuda_dev, x, u=u, pos=pos) == want(x, [1.0] * 4, [0] * 4, [1.0] * 4, [0.0] * 4, u)
    assert int(pos) == 42
    tok = torch.empty(4, dtype=torch.int64, device=cuda_dev)
    ext().argmax_next(x.bfloat16()[:, :496].contiguous().to(cuda_dev), tok)
    assert draw(cuda_dev, x.bfloat16()[:, :496], temperature=[0.0] * 4, u=u) == tok.cpu().tolist()


def test_distribution(cuda_dev):
    """Evenly spaced uniforms give every token its share, to one draw."""
    x = torch.tensor([[0.0, 1.0, 2.0, -1.0, 0.5]])
    n = 4000
    toks = draw(cuda_dev, x.expand(n, 5).contiguous(), u=((np.arange(n) + 0.5) / n).tolist())
    share = torch.softmax(x[0].double(), 0) * n
    for i in range(5):
        assert abs(toks.count(i) - share[i].item()) <= 1.0


def test_capture_and_refusals(cuda_dev):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(3, 2000, generator=g).to(cuda_dev)
    u, tok = torch.rand(3, device=cuda_dev), torch.zeros(3, dtype=torch.int64, device=cuda_dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ext().sample_next(x, None, None, None, None, u, tok)
    x.copy_(torch.randn(3, 2000, generator=g).to(cuda_dev))
    graph.replay()
    assert tok.cpu().tolist() == want(x, [1.0] * 3, [0] * 3, [1.0] * 3, [0.0] * 3, u.cpu().tolist())
    K = ext()
    K.sample_next(x[:0], None, None, None, None, u[:0], tok[:0])
    for args, match in (((x.double(), None, None, None, None, u, tok), "logits"),
                        ((x.t(), None, None, None, None, u, tok), "logits"),
                        ((x, u[:2], None, None, None, u, tok), "temperature"),
                        ((x, None, u, None, None, u, tok), "top_k"), ((x, None, None, None, None, None, tok), "u:"),
                        ((x, None, None, None, None, u, tok.int()), "tok"),
                        ((torch.zeros(3, (1 << 18) + 1, device=cuda_dev), None, None, None, None, u, tok), "262144")):
        with pytest.raises(RuntimeError, match=match):
            K.sample_next(*args)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
def test_extreme_parameters(cuda_dev, dt):
    """Temperatures next to zero and infinite ones, uniforms at and past their ends, spreads beyond every bin."""
    g = torch.Generator().manual_seed(7)
    base = 3 * torch.randn(2500, generator=g)
    rows, p = [], dict(temperature=[], top_k=[], top_p=[], min_p=[], u=[])
    for T in (1e-45, 1e-38, 1e-30, 1e-20, 1e-3, 1e20, 3e38, float("inf")):
        for k, tp in ((0, 1.0), (0, 0.5), (40, 1.0), (40, 0.5), (2400, 0.999)):
            for u in (0.0, 0.5, 1.0, 1.5, -1.0, float("nan")):
                rows.append(base)
                for n, v in zip(p, (T, k, tp, 0.0, u)):
                    p[n].append(v)
    x = torch.stack(rows).to(DT[dt])
    assert draw(cuda_dev, x, **p) == want(x, **p)


@pytest.mark.parametrize("scale", [1e-30, 1e-6, 0.01, 1.0, 30.0, 3000.0])
def test_spreads(cuda_dev, scale):
    """Cuts in distributions from flat (thousands of elements in a bin) to a single spike."""
    g = torch.Generator().manual_seed(8)
    x = scale * torch.randn(30, 20000, generator=g)
    p = params(np.random.default_rng(8), 30)
    p["temperature"] = [1.0] * 30
    assert draw(cuda_dev, x, **p) == want(x, **p)


@pytest.mark.parametrize("dt", ["bf16", "fp32"])
@pytest.mark.parametrize("k", [2, 3, 31, 100, 127, 128, 129, 130, 300])
def test_lists_on_both_sides_of_the_pairwise_limit(cuda_dev, k, dt):
    """top_k around 128, with ties across the cut (equal logits at the k-th place) and without, each filter on and off."""
    g = torch.Generator().manual_seed(k)
    B, V = 24, 30011
    x = 2.0 * torch.randn(B, V, generator=g)
    x[::3] = (x[::3] * 4).round() / 4  # many equal logits
    x = x.to(DT[dt])
    rng = np.random.default_rng(k)
    pick = lambda *a: [a[i % len(a)] for i in range(B)]  # noqa: E731
    p = dict(temperature=pick(0.5, 1.0, 1.0, 2.0, 1e-4), top_k=[k] * B, top_p=pick(1.0, 0.9, 0.3, 0.99),
             min_p=pick(0.0, 0.0, 0.2, 0.0, 0.01), u=rng.random(B, dtype=np.float32).tolist())
    p["u"][:2] = [0.0, float(np.nextafter(np.float32(1), np.float32(0)))]
    assert draw(cuda_dev, x, **p) == want(x, **p)


@pytest.mark.parametrize("dt", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("B,V", [(1, 65536), (20, 5000), (200, 65536)])
def test_flat_tails_at_the_last_bins(cuda_dev, B, V, dt):
    """Thousands of equal logits 45.9 binary orders below the largest (1022 of 1024 bins, 46 orders in all), where the
    counted elements end, with a top_k or a nucleus whose cut lies there: what is counted is what is listed."""
    bins = 1024 / (46 * np.log(2))  # bins a unit of logits at temperature 1
    places = (1020.6, 1021.4, 1021.6, 1021.9, 1022.1, 1022.4, 1022.6, 1023.4)
    x = torch.full((B, V), -64.0)
    x[:, 0] = 0.0
    x[1::2, V // 2] = -63.97  # half a bin above the others, where the type holds it
    p = dict(temperature=[float(64.0 * bins / places[b % 8]) for b in range(B)],
             top_k=[(0, 2, 0, 3, 0, 2, 2000)[b % 7] for b in range(B)],
             top_p=[(1 - 2**-18, 1.0, 0.99999, 0.999999, 1 - 2**-20)[b % 5] for b in range(B)],
             min_p=[0.0] * B, u=[(0.3, 0.999999, 1.0, 0.0)[b % 4] for b in range(B)])
    if B == 1:
        p.update(top_p=[0.99999], temperature=[float(64.0 * bins / 1022.2)])
    assert draw(cuda_dev, x.to(DT[dt]), **p) == want(x.to(DT[dt]), **p)


@pytest.mark.parametrize("ties", [60, 1500])
def test_ties_between_two_bins(cuda_dev, ties):
    """Equal logits whose place lies so near the border of two of the 1024 bins that it depends on whether a product is
    rounded before a sum: every pass puts them into the same one, so the cut's list is complete."""
    f = np.float32
    scale = f(f(np.log2(np.e) * 1024 / 46))
    v = np.random.default_rng(0).uniform(1.0, 20.0, 1 << 22).astype(f)
    place = (v * scale).astype(f)
    once = (v.astype(np.float64) * np.float64(scale) + 2.0**23).astype(f)  # the product unrounded
    v = v[once != (place + f(2.0**23)).astype(f)][:40]
    assert len(v) == 40
    g = torch.Generator().manual_seed(ties)
    x = -24.0 - torch.rand(len(v), 5000, generator=g)
    x[:, 100:120] = -torch.rand(len(v), 20, generator=g)
    x[:, 7] = 0.0
    x[:, 2000:2000 + ties] = -torch.from_numpy(v)[:, None]
    rng = np.random.default_rng(ties)
    B = len(v)
    p = dict(temperature=[1.0] * B, top_k=[(0, 50, 22, 21 + ties)[b % 4] for b in range(B)],
             top_p=[(0.9, 1.0, 0.99999, 1.0, 0.5)[b % 5] for b in range(B)], min_p=[0.0] * B,
             u=rng.random(B, dtype=f).tolist())
    p["u"][::3] = [0.99999] * len(p["u"][::3])
    assert draw(cuda_dev, x, **p) == want(x, **p)


def test_spreads_past_the_largest_float(cuda_dev):
    """Differences of fp32 logits beyond 3.4e38, at temperatures where they still weigh."""
    g = torch.Generator().manual_seed(9)
    base = 3.4e38 * (2 * torch.rand(3000, generator=g) - 1)
    rows, p = [], dict(temperature=[], top_k=[], top_p=[], min_p=[], u=[])
    for T in (1e37, 1e38, 3.4e38, float("inf")):
        for k, tp, mp in ((0, 1.0, 0.0), (0, 1.0, 0.2), (0, 0.9, 0.0), (0, 0.5, 0.1), (2000, 1.0, 0.0), (50, 0.9, 0.0)):
            for u in (0.0, 0.3, 0.6, 0.999):
                rows.append(base)
                for n, v in zip(p, (T, k, tp, mp, u)):
                    p[n].append(v)
    x = torch.stack(rows)
    assert draw(cuda_dev, x, **p) == want(x, **p)
