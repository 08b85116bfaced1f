"""The paged cache's two bookkeeping operators on the B200: block tables and slot maps (kv_slots, whole numbers, equal
to the definition) and q/k norm + rotary positions + cache write (qk_norm_rope_kv_paged, against 64 bits).

Tolerance of the rotary kernel, from its arithmetic: one rounding to the type (half a step, eps / 2 relative) of a value
computed in fp32 from two products: the angle is exact to about 1e-7 (its fp32 reduced value, |r| <= pi, is off by at
most 1.2e-7, cos and sin by as much again), the norm and the two products add a few 2^-24. So |err| <= eps / 2 |y| +
1e-6 (|x_a| + |x_b|), and the pair is bounded by the head's largest value times sqrt(D) under the norm.
"""

import numpy as np
import pytest
import torch

from lfm2opt.kernels import ext
from lfm2opt.rope import inv_freq
from oracle.serving import kv_slots_ref, rope_paged_f64

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ---------------------------------------------------------------------------------------------------- kv_slots
class Pool:
    """The device state of kv_slots and, beside it, the definition's."""

    def __init__(self, B, width, pages, page, capacity, dev, seed=0):
        rng = np.random.default_rng(seed)
        self.page, self.capacity, self.dev, self.B = page, capacity, dev, B
        self.free = rng.permutation(pages).astype(np.int32)
        self.n_free, self.table = pages, np.full((B, width), -1, np.int32)
        self.lens = np.zeros(B, np.int32)
        i32 = lambda a: torch.from_numpy(np.array(a, np.int32)).to(dev)  # noqa: E731
        self.d_free, self.d_n, self.d_table = i32(self.free), i32([pages]), i32(self.table)

    def step(self, want):
        """One call on both; asserts equality of everything and returns got."""
        want = np.asarray(want, np.int32)
        got, cu, pos, slots, self.table, self.free, self.n_free = kv_slots_ref(
            self.lens, want, self.table, self.free, self.n_free, self.page, self.capacity)
        d_got = torch.full((self.B,), -7, dtype=torch.int32, device=self.dev)
        d_cu = torch.full((self.B + 1,), -7, dtype=torch.int32, device=self.dev)
        d_pos = torch.full((self.capacity,), -7, dtype=torch.int64, device=self.dev)
        d_slots = torch.full_like(d_pos, -7)
        ext().kv_slots(torch.from_numpy(self.lens).to(self.dev), torch.from_numpy(want).to(self.dev), self.d_table,
                       self.d_free, self.d_n, self.page, d_got, d_cu, d_pos, d_slots)
        n = len(pos)
        assert np.array_equal(d_got.cpu(), got) and np.array_equal(d_cu.cpu(), cu)
        assert np.array_equal(d_pos[:n].cpu(), pos) and np.array_equal(d_slots[:n].cpu(), slots)
        assert (d_pos[n:] == -7).all() and (d_slots[n:] == -7).all()  # rows behind the last token: as they were
        assert np.array_equal(d_table_cpu(self.d_table), self.table)
        assert int(self.d_n) == self.n_free and np.array_equal(self.d_free.cpu()[:self.n_free], self.free[:self.n_free])
        self.lens = got.astype(np.int32)
        return got


def d_table_cpu(t):
    return t.cpu().numpy()


@pytest.mark.parametrize("B,width,pages,page,capacity", [
    (1, 1, 1, 1, 1), (3, 5, 8, 16, 40), (37, 64, 900, 16, 4096), (64, 20, 1100, 64, 70000), (1000, 9, 3000, 7, 5000),
    (1025, 4, 2500, 32, 30000), (2500, 3, 4000, 24, 9000)])
def test_kv_slots_follows_the_definition_over_a_life(cuda_dev, B, width, pages, page, capacity):
    """Admissions, growth, shrinking and ends, more wanted than the pool or the token rows hold."""
    p = Pool(B, width, pages, page, capacity, cuda_dev, seed=B)
    rng = np.random.default_rng(B + 1)
    room = width * page
    p.step(rng.integers(0, room + 1, B))
    p.step(p.lens + rng.integers(0, 2 * page, B) * (rng.random(B) < 0.5))
    p.step(np.where(rng.random(B) < 0.3, 0, p.lens))  # some end
    p.step(np.clip(p.lens + rng.integers(-page, page + 1, B), -1, room + 3))  # lengths out of range are refused
    p.step(np.zeros(B))
    assert p.n_free == pages and sorted(p.d_free.cpu().tolist()) == list(range(pages))


def test_kv_slots_growing_and_shrinking_back_restores_the_stack(cuda_dev):
    p = Pool(50, 40, 1500, 16, 8192, cuda_dev)
    base = p.step(np.arange(50) * 9)
    before = p.d_free.clone(), p.d_table.clone()
    p.step(base + 33)
    p.step(base)
    assert torch.equal(p.d_free, before[0]) and torch.equal(p.d_table, before[1])


def test_kv_slots_empty_batch_and_refused_requests(cuda_dev):
    p = Pool(4, 4, 5, 8, 64, cuda_dev)
    assert p.step([8, 33, 8, 0]).tolist() == [8, 0, 8, 0]      # 33 > 4 pages of 8: refused, and takes nothing
    assert p.step([32, 0, 24, 0]).tolist() == [32, 0, 8, 0]    # three pages of five for the first, none for the third
    z = torch.zeros(0, dtype=torch.int32, device=cuda_dev)
    cu = torch.full((1,), 9, dtype=torch.int32, device=cuda_dev)
    ext().kv_slots(z, z, torch.zeros(0, 4, dtype=torch.int32, device=cuda_dev), p.d_free, p.d_n, 8, z.clone(), cu,
                   torch.zeros(0, dtype=torch.int64, device=cuda_dev), torch.zeros(0, dtype=torch.int64, device=cuda_dev))
    assert int(cu) == 0 and int(p.d_n) == p.n_free


@pytest.mark.parametrize("each,got", [(1 << 29, [1 << 29, 1 << 29, 0, 0]), ((1 << 29) + 1, [(1 << 29) + 1, 0, 0, 0])])
def test_kv_slots_at_the_largest_capacity(cuda_dev, each, got):
    """2^30 token rows (16 GB): two requests that fill them to the last, and two that together bring two more."""
    page, cap = 1 << 20, 1 << 30
    i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=cuda_dev)  # noqa: E731
    table = torch.full((4, 1024), -1, dtype=torch.int32, device=cuda_dev)
    free, n_free = torch.arange(1500, dtype=torch.int32, device=cuda_dev), i32([1500])
    d_got, cu = i32([-7] * 4), i32([-7] * 5)
    pos, slots = [torch.full((cap,), -7, dtype=torch.int64, device=cuda_dev) for _ in range(2)]
    ext().kv_slots(i32([0] * 4), i32([each, each, 5, 0]), table, free, n_free, page, d_got, cu, pos, slots)
    cut = np.cumsum([0] + got)
    assert d_got.tolist() == got and cu.tolist() == cut.tolist()
    pages = [-(-g // page) for g in got]
    assert int(n_free) == 1500 - sum(pages) and [int((r >= 0).sum()) for r in table] == pages
    for b, n in enumerate(got):
        for t0 in range(0, n, 1 << 28):  # in pieces: a comparison makes several copies
            t = torch.arange(t0, min(n, t0 + (1 << 28)), device=cuda_dev)
            at = slice(int(cut[b]) + t0, int(cut[b]) + t0 + len(t))
            assert torch.equal(pos[at], t)
            assert torch.equal(slots[at], table[b, t // page].long() * page + t % page)
    assert (pos[cut[-1]:] == -7).all() and (slots[cut[-1]:] == -7).all()


# ---------------------------------------------------------------------------------------------------- rotary positions
@pytest.mark.parametrize("N,NQ,NKV,D,rot,inter,norm,dt,page,far,kind", [
    (1, 32, 8, 64, 64, False, True, "bf16", 64, 4000, "plain"),
    (5, 1, 1, 64, 16, True, False, "fp16", 1, 10, "plain"),
    (7, 24, 3, 128, 64, False, True, "fp16", 16, 131072, "yarn"),
    (9, 5, 5, 128, 128, True, True, "bf16", 24, 1000000, "llama3"),
    (33, 8, 2, 64, 32, False, False, "bf16", 5, 2**31 + 5, "ntk"),
    (3, 64, 8, 128, 128, False, True, "fp16", 64, 2**24, "linear"),
    (2, 300, 1, 64, 48, False, True, "bf16", 64, 77, "plain"),
])
def test_rope_paged_against_64_bits(cuda_dev, N, NQ, NKV, D, rot, inter, norm, dt, page, far, kind):
    g = torch.Generator().manual_seed(N * NQ + D)
    T = DT[dt]
    pages = -(-N // page) + 2
    wide = torch.randn(N, (NQ + 2 * NKV) * D + 24, generator=g).to(T)  # rows further apart than they are long
    qkv = wide[:, 8:8 + (NQ + 2 * NKV) * D]
    kc, vc = torch.randn(pages, NKV, page, D, generator=g).to(T), torch.randn(pages, NKV, page, D, generator=g).to(T)
    qw, kw = [(torch.rand(D, generator=g) + 0.5).to(T) if norm else None for _ in range(2)]
    f, scaling = inv_freq(rot, kind=kind, factor=4.0 if kind != "plain" else 1.0, original=8192)
    positions = torch.randint(0, far, (N,), generator=g)
    slots = torch.randperm(pages * page, generator=g)[:N]
    if N > 2:
        slots[1], slots[2] = -1, pages * page  # padding, and a slot behind the pool: neither is written
    want = rope_paged_f64(qkv, qw, kw, f, scaling, positions, slots, kc, vc, NQ, 1e-5, inter)
    d = lambda t: None if t is None else t.to(cuda_dev)  # noqa: E731
    dq = d(wide)[:, 8:8 + (NQ + 2 * NKV) * D]
    q, dk, dv = torch.full((N, NQ, D), float("nan"), dtype=T, device=cuda_dev), d(kc), d(vc)
    ext().qk_norm_rope_kv_paged(dq, d(qw), d(kw), d(f), scaling, d(positions), d(slots), q, dk, dv, 1e-5, inter)
    # |x_a| + |x_b| of a pair, normed: at most 1.5 sqrt(D) (a head of norm sqrt(D)) each, else the inputs' largest
    big = scaling * 2 * (1.5 * D ** 0.5 if norm else qkv.float().abs().max().item())
    for got, ref in ((q, want[0]), (dk, want[1]), (dv, want[2])):
        err = (got.cpu().double() - ref).abs()
        assert (err <= torch.finfo(T).eps / 2 * ref.abs() + 1e-6 * big).all(), err.max().item()
    assert torch.equal(dv.cpu().double(), want[2])  # values keep their bits


def test_rope_paged_empty_and_refusals(cuda_dev):
    K = ext()
    e = dict(dtype=torch.bfloat16, device=cuda_dev)
    kc, vc = torch.zeros(2, 1, 16, 64, **e), torch.zeros(2, 1, 16, 64, **e)
    f = inv_freq(64, device=cuda_dev)[0]
    i = lambda n: torch.zeros(n, dtype=torch.int64, device=cuda_dev)  # noqa: E731
    K.qk_norm_rope_kv_paged(torch.zeros(0, 192, **e), None, None, f, 1.0, i(0), i(0), torch.zeros(0, 1, 64, **e), kc, vc,
                            1e-5)
    q, x = torch.zeros(1, 1, 64, **e), torch.zeros(1, 192, **e)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        K.qk_norm_rope_kv_paged(x, None, None, f[:4], 1.0, i(1), i(1), q, kc, vc, 1e-5)
    with pytest.raises(RuntimeError, match="both or neither"):
        K.qk_norm_rope_kv_paged(x, q[0, 0], None, f, 1.0, i(1), i(1), q, kc, vc, 1e-5)
    with pytest.raises(RuntimeError, match="dtype"):
        K.qk_norm_rope_kv_paged(x.half(), None, None, f, 1.0, i(1), i(1), q, kc, vc, 1e-5)
    with pytest.raises(RuntimeError, match="NQ"):
        K.qk_norm_rope_kv_paged(x[:, :128].contiguous(), None, None, f, 1.0, i(1), i(1), q, kc, vc, 1e-5)
