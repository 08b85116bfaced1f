"""The batched-serving operators without a GPU: refusals of the C ABI come before the device, the frequency tables
follow their formulas, and the plain forms agree with direct ones."""

import math

import numpy as np
import pytest
import torch

from lfm2opt import _capi
from lfm2opt.rope import inv_freq
from oracle.serving import kv_slots_ref, sample_next_f64, tree_attention_f64

F = 1 << 20  # 16-byte aligned, never dereferenced


def refused(name, args, match):
    st = getattr(_capi.lib(), name)(*args)
    assert st == _capi.EINVAL, st
    assert match in _capi.lib().lfm2q_last_error().decode(), _capi.lib().lfm2q_last_error()


def swap(args, **at):
    a = list(args)
    for k, v in at.items():
        a[int(k[1:])] = v
    return a


def test_kv_slots_refusals():
    ok = [F, F + 64, F, F, F, F + 128, F, F, F, 4, 8, 100, 16, 64, None]
    for at, match in ((dict(_9=-1), "B >= 0"), (dict(_10=0), "max_pages"), (dict(_11=0), "num_pages"),
                      (dict(_12=0), "page"), (dict(_10=1 << 27), "2^30"), (dict(_13=-1), "capacity"),
                      (dict(_2=None), "non-null"), (dict(_5=F + 64), "got"), (dict(_5=F), "got")):
        refused("lfm2q_kv_slots", swap(ok, **at), match)


def test_rope_refusals():
    ok = [F, 1024, F, F, F, 64, 1.0, F, F, F, F, F, _capi.BF16, 4, 8, 4, 64, 10, 16, 1e-5, 0, None]
    for at, match in ((dict(_12=_capi.FP32), "dtype"), (dict(_16=96), "head_dim"), (dict(_5=8), "rot_dim"),
                      (dict(_5=80), "rot_dim"), (dict(_1=1016), "stride"), (dict(_1=1028), "stride"),
                      (dict(_2=None), "both or neither"), (dict(_0=F + 8), "aligned"), (dict(_13=-1), "N >= 0"),
                      (dict(_7=None), "non-null")):
        refused("lfm2q_qk_norm_rope_kv_paged", swap(ok, **at), match)
    assert _capi.lib().lfm2q_qk_norm_rope_kv_paged(*swap(ok, _13=0)) == _capi.OK


def test_tree_attention_refusals():
    ok = [F] * 9 + [_capi.BF16, 20, 2, 8, 2, 64, 10, 16, 8, 2, 10, 0.125, None]
    for at, match in ((dict(_9=7), "dtype"), (dict(_14=80), "head_dim"), (dict(_12=9), "multiple of NKV"),
                      (dict(_12=130), "64 times"), (dict(_19=0), "max_q"), (dict(_19=65), "max_q"),
                      (dict(_18=0), "S <="), (dict(_20=0.0), "scale"), (dict(_20=float("nan")), "scale"),
                      (dict(_8=None), "ws"), (dict(_0=F + 2), "aligned"), (dict(_17=1 << 27), "2^30"),
                      (dict(_11=70000), "65535"), (dict(_5=None), "non-null")):
        refused("lfm2q_tree_attention", swap(ok, **at), match)
    assert _capi.lib().lfm2q_tree_attention(*swap(ok, _10=0)) == _capi.OK
    assert _capi.lib().lfm2q_tree_attention_splits(0, 8, 2, 64, 1, 100) == 1
    assert 1 <= _capi.lib().lfm2q_tree_attention_splits(1, 32, 8, 64, 1, 100000) <= 64


def test_tree_attention_refuses_more_tiles_than_its_line_holds():
    """B * NKV * ceil(max_q G / (whole queries of 128 rows)) * (max_pages * page / 64 + 8) < 2^31 - 2^16"""
    ok = [F] * 9 + [_capi.BF16, 20, 1024, 32, 32, 64, 10, 64, 65000, 2, 1, 0.125, None]
    refused("lfm2q_tree_attention", swap(ok, _17=65536), "2^31")  # 1024 * 32 * (65536 + 8)
    # two queries a tile: five take three, 512 * 32 * 3 * 65008 (three take two, 2^31 - 17301504)
    refused("lfm2q_tree_attention", swap(ok, _11=512, _12=32 * 64, _19=5), "2^31")
    for at in (dict(), dict(_11=512, _12=32 * 64, _19=3), dict(_11=512, _12=32 * 64, _19=1)):
        st = _capi.lib().lfm2q_tree_attention(*swap(ok, **dict(at, _10=0)))  # N = 0: checked, nothing to do
        assert st == _capi.OK, _capi.lib().lfm2q_last_error()


def test_sample_refusals():
    ok = [F, _capi.BF16, 1000, None, None, None, None, F, F, None, 2, 1000, None]
    for at, match in ((dict(_1=3), "dtype"), (dict(_2=999), "stride"), (dict(_11=0), "V <="),
                      (dict(_11=1 << 19, _2=1 << 19), "V <="), (dict(_10=70000), "65535"), (dict(_7=None), "non-null"),
                      (dict(_0=F + 1), "aligned")):
        refused("lfm2q_sample_next", swap(ok, **at), match)
    assert _capi.lib().lfm2q_sample_next(*swap(ok, _10=0)) == _capi.OK


@pytest.mark.skipif(torch.cuda.is_available(), reason="checks the no-device path")
def test_valid_calls_without_a_device_are_not_supported():
    assert _capi.lib().lfm2q_sample_next(F, 0, 1000, None, None, None, None, F, F, None, 2, 1000, None) == _capi.ENOTSUP
    assert _capi.lib().lfm2q_kv_slots(F, F + 64, F, F, F, F + 128, F, F, F, 4, 8, 100, 16, 64, None) == _capi.ENOTSUP


def test_frequency_tables():
    base, s = inv_freq(64, 1e6)
    i = np.arange(32)
    assert s == 1.0 and base.dtype == torch.float32
    assert np.array_equal(base.numpy(), (1e6 ** (-2.0 * i / 64)).astype(np.float32))
    assert torch.equal(inv_freq(64, 1e6, "linear", 4.0)[0], base / 4)
    ntk = inv_freq(64, 1e6, "ntk", 4.0)[0].double().numpy()
    assert ntk[0] == 1.0 and abs(ntk[-1] * 4 / base[-1].item() - 1) < 1e-6
    yarn, s = inv_freq(128, 1e4, "yarn", 16.0, original=4096)
    plain = inv_freq(128, 1e4)[0]
    turns = 4096 * plain.double() / (2 * math.pi)
    assert abs(s - (0.1 * math.log(16) + 1)) < 1e-12
    assert torch.equal(yarn[turns > 40], plain[turns > 40])
    assert torch.allclose(yarn[turns < 0.8], plain[turns < 0.8] / 16, rtol=1e-6)
    ll = inv_freq(128, 5e5, "llama3", 8.0, original=8192)[0]
    plain = inv_freq(128, 5e5)[0]
    turns = 8192 * plain.double() / (2 * math.pi)
    assert torch.equal(ll[turns >= 4], plain[turns >= 4])
    assert torch.allclose(ll[turns <= 1], plain[turns <= 1] / 8, rtol=1e-6)
    mid = (turns > 1) & (turns < 4)
    w = (turns[mid] - 1) / 3
    assert torch.allclose(ll[mid].double(), plain[mid].double() * (w + (1 - w) / 8), rtol=1e-6)
    for bad in (dict(rot_dim=7), dict(rot_dim=64, factor=0.5), dict(rot_dim=64, kind="yarn", factor=2.0),
                dict(rot_dim=64, kind="other")):
        with pytest.raises(ValueError):
            inv_freq(**bad)


def test_plain_forms_agree_with_direct_ones():
    rng = np.random.default_rng(0)
    # one request, every position seen: plain softmax attention
    q, k, v = torch.randn(1, 2, 64), torch.randn(4, 1, 8, 64), torch.randn(4, 1, 8, 64)
    out = tree_attention_f64(q, k, v, torch.tensor([[2, 0, 3, 1]]), [20], [0, 1], None, 0.125)
    kk, vv = [t[[2, 0, 3, 1], 0].reshape(-1, 64)[:21].double() for t in (k, v)]
    assert torch.allclose(out[0], torch.softmax(q[0].double() @ kk.T * 0.125, -1) @ vv)
    # growth hands out pages from the top of the stack
    got, cu, pos, slots, table, free, top = kv_slots_ref(np.array([3]), np.array([6]), np.array([[7, -1]]),
                                                         np.array([1, 5]), 2, 4, 10)
    assert (got.tolist(), cu.tolist(), pos.tolist(), slots.tolist(), table.tolist(), top) == \
        ([6], [0, 3], [3, 4, 5], [31, 20, 21], [[7, 5]], 1)
    x = rng.normal(size=100)
    p = np.exp(x - x.max())
    assert sample_next_f64(x, 1.0, 0, 1.0, 0.0, 0.5) == int(np.searchsorted(np.cumsum(p), 0.5 * p.sum(), side="right"))
    assert sample_next_f64(x, 1.0, 1, 1.0, 0.0, 0.99) == int(x.argmax())


@pytest.mark.skipif(torch.cuda.is_available(), reason="some of the calls are valid but for their pointers")
def test_arguments_in_one_block():
    """lfm2q_call_words: the same answer as the entry point for each operator, and its own refusals."""
    L = _capi.lib()
    calls = {_capi.KV_SLOTS: ("lfm2q_kv_slots", [F, F + 64, F, F, F, F + 128, F, F, F, 4, 8, 100, 16, 64, 0], 12),
             _capi.QK_NORM_ROPE_KV_PAGED: ("lfm2q_qk_norm_rope_kv_paged",
                                           [F, 1024, F, F, F, 64, 1.0, F, F, F, F, F, _capi.BF16, 4, 8, 4, 64, 10, 16,
                                            1e-5, 0, 0], 5),
             _capi.TREE_ATTENTION: ("lfm2q_tree_attention",
                                    [F] * 9 + [_capi.BF16, 20, 2, 8, 2, 64, 10, 16, 8, 2, 10, 0.125, 0], 19),
             _capi.SAMPLE_NEXT: ("lfm2q_sample_next", [F, _capi.BF16, 1000, 0, 0, 0, 0, F, F, 0, 2, 1000, 0], 11)}
    for (code, pack, n), (name, ok, number) in calls.items():
        assert len(ok) == n == len(_capi.SIGNATURES[name])
        kinds = [type(v) for v in ok]
        for k in range(n):  # every argument in its place: a bad value of each is answered alike
            for bad in ((-1.0, float("nan")) if kinds[k] is float else (0, 7, -5)):
                a = swap(ok, **{f"_{k}": bad})
                st = getattr(L, name)(*[None if v == 0 and t is _capi._p else v
                                        for v, t in zip(a, _capi.SIGNATURES[name])])
                said = L.lfm2q_last_error()
                assert L.lfm2q_call_words(code, pack(*a), n) == st, (name, k, bad)
                assert L.lfm2q_last_error() == said, (name, k, bad)
        refused("lfm2q_call_words", (code, pack(*ok), n - 1), "number of arguments")
        refused("lfm2q_call_words", (code, pack(*swap(ok, **{f"_{number}": 1 << 32})), n), "32 bits")
    refused("lfm2q_call_words", (4, bytes(8 * 24), 13), "no such operator")
    refused("lfm2q_call_words", (0, None, 15), "number of arguments")


@pytest.mark.parametrize("kind", ["BatchDecodeStep", "DecodeStep"])
def test_a_step_is_captured_on_its_own_device(monkeypatch, kind):
    """Without a stream torch.cuda.graph captures on one of the device that was current at the process's first capture;
    the step's launches go to streams of the weights' device, and would run at once in place of being captured."""
    import contextlib
    from types import SimpleNamespace

    from lfm2opt import batch_step, decode_step
    dev, current, seen = torch.device("cuda", 1), [None], []

    class Stream:
        def __init__(self, device=None):
            self.device = device

        def wait_stream(self, other):
            assert other.device == self.device == dev

    @contextlib.contextmanager
    def use(stream):
        old, current[0] = current[0], stream
        yield
        current[0] = old

    def graph(g, stream=None, **kw):
        return use(stream if stream is not None else Stream(torch.device("cuda", 0)))

    for name, fake in (("Stream", Stream), ("current_stream", Stream), ("stream", use), ("graph", graph),
                       ("CUDAGraph", object)):
        monkeypatch.setattr(torch.cuda, name, fake)
    cls = getattr(batch_step if kind == "BatchDecodeStep" else decode_step, kind)
    s = object.__new__(cls)
    s.h, s.active = SimpleNamespace(device=dev), torch.ones(2, dtype=torch.int32)
    s.step = lambda: seen.append(current[0].device)
    assert s.capture() is s
    assert seen == [dev, dev] and s.active.tolist() == [1, 1]
