"""The batched decode step (lfm2opt.batch_step.BatchDecodeStep): kv_slots, qk_norm_rope_kv_paged, tree_attention and
sample_next run together as a serving loop runs them.

On contexts of one tile, where a request's arithmetic does not depend on its neighbours (the GEMMs' integer sums are
exact, the attention is not split), a request in a batch gives the same bits as alone, whatever page it got and whoever
came and went beside it. Longer contexts and the whole step are compared with a plain fp32 form of it.
"""

import pytest
import torch
import torch.nn.functional as F

from lfm2opt.batch_step import BatchDecodeStep
from lfm2opt.decode_step import Lfm2Config, Lfm2Weights

pytestmark = pytest.mark.gpu
CFG = Lfm2Config(hidden=512, layers=4, attn_layers=(1, 3), n_heads=8, n_kv=2, inter=1024, vocab=1000)


@pytest.fixture(scope="module")
def weights(cuda_dev):
    return Lfm2Weights(CFG, cuda_dev, seed=3)


def alone(weights, toks):
    """Logits of every position of one request fed `toks`, in a step of its own."""
    s, out = BatchDecodeStep(weights, 1, 4, page=16, max_pages=4), []
    s.active.fill_(1)
    for t in toks:
        s.tok.fill_(t)
        s.step()
        out.append(s.logits[0].clone())
    return torch.stack(out)


def plain(weights, toks):
    """The same step in fp32 torch operations, one sequence; linears on the quantized weights and inputs."""
    c = weights.cfg
    bf = lambda t: t.to(torch.bfloat16).float()  # noqa: E731

    def norm(x, w):
        return bf(w.float() * bf(x * torch.rsqrt(x.square().mean(-1, keepdim=True) + c.eps)))

    def lin(x, wq):
        s = x.abs().amax(-1, keepdim=True).clamp_min(1e-8) / 127
        return bf((torch.round(x / s) @ wq[0].float().T) * s * wq[1])

    h = weights.embed[toks].float()
    n = len(toks)
    for i, L in enumerate(weights.layer):
        x = norm(h, weights.norm[i])
        if i in c.attn_layers:
            q, k, v = lin(x, L["qkv"]).view(n, -1, c.head_dim).split([c.n_heads, c.n_kv, c.n_kv], 1)
            ang = torch.arange(n, device=h.device)[:, None] * weights.inv_freq
            cos, sin = torch.cat([ang.cos()] * 2, -1)[:, None], torch.cat([ang.sin()] * 2, -1)[:, None]

            def turn(t, w):
                t = t * torch.rsqrt(t.square().mean(-1, keepdim=True) + c.eps) * w.float()
                a, b = t.chunk(2, -1)
                return bf(t * cos + torch.cat([-b, a], -1) * sin)

            q, k = turn(q, L["qw"]).transpose(0, 1), turn(k, L["kw"]).transpose(0, 1)
            k, v = [t.repeat_interleave(c.n_heads // c.n_kv, 0) for t in (k, v.transpose(0, 1))]
            s = (q @ k.transpose(1, 2)) * c.head_dim ** -0.5
            s = s.masked_fill(torch.ones(n, n, device=h.device).triu(1) > 0, float("-inf"))
            y = lin(bf((s.softmax(-1) @ v).transpose(0, 1).reshape(n, -1)), L["o"])
        else:
            b, cc, xx = lin(x, L["in"]).chunk(3, -1)
            bx = F.pad(bf(b * xx), (0, 0, 2, 0))
            w = L["cw"].float()
            y = lin(bf(cc * bf(bx[:-2] * w[:, 0] + bx[1:-1] * w[:, 1] + bx[2:] * w[:, 2])), L["out"])
        h = bf(h + y)
        g, u = lin(norm(h, weights.ffn_norm[i]), L["w13"]).chunk(2, -1)
        h = bf(h + lin(bf(bf(F.silu(g)) * u), L["w2"]))
    return lin(norm(h, weights.norm[-1]), weights.head)


def test_requests_in_a_batch_equal_requests_alone(cuda_dev, weights):
    """Five request slots, a pool too small for all to be long: requests come, go, wait for a page and go on."""
    g = torch.Generator().manual_seed(1)
    feeds = [torch.randint(0, CFG.vocab, (n,), generator=g).tolist() for n in (40, 25, 33, 17, 9)]
    want = [alone(weights, f) for f in feeds]
    s = BatchDecodeStep(weights, 5, 6, page=16, max_pages=4)  # 3 + 2 + 3 + 2 + 1 pages would be needed at once
    done, fed, waited = [False] * 5, [0] * 5, 0
    for it in range(200):
        if all(done):
            break
        s.active.copy_(torch.tensor([int(not done[b] and it >= 3 * b) for b in range(5)]))
        s.tok.copy_(torch.tensor([feeds[b][min(fed[b], len(feeds[b]) - 1)] for b in range(5)]))
        before = s.lens.clone()
        s.step()
        grew = (s.lens - before).tolist()
        for b in range(5):
            if grew[b]:
                assert torch.equal(s.logits[b], want[b][fed[b]]), (it, b, fed[b])
                fed[b] += 1
            elif s.active[b]:
                waited += 1
            if fed[b] == len(feeds[b]) and not done[b]:
                done[b] = True
                s.release(b)
    assert all(done) and waited > 0
    assert int(s.n_free) == 6 and sorted(s.free.tolist()) == list(range(6)) and int(s.table.max()) == -1


def test_step_against_a_plain_form(cuda_dev, weights):
    """150 positions over pages in use by others: several tiles, split attention. Both round to bf16 at the same places;
    a last-bit difference of an activation moves its int8 code by at most one, so the bar is that of the other
    whole-stack comparisons: max |err| <= 5e-2, mean |err| <= 1e-2 of the largest logit."""
    g = torch.Generator().manual_seed(2)
    toks = torch.randint(0, CFG.vocab, (150,), generator=g).to(cuda_dev)
    s = BatchDecodeStep(weights, 3, 40, page=8, max_pages=24)
    s.active.copy_(torch.tensor([1, 1, 0]))
    out = []
    for n in range(150):
        s.tok[0], s.tok[1] = toks[n], toks[149 - n]
        s.step()
        out.append(s.logits[:2].float())
    out = torch.stack(out)
    for b, t in ((0, toks), (1, toks.flip(0))):
        ref = plain(weights, t)
        err, m = (out[:, b] - ref).abs(), ref.abs().max()
        assert err.max() <= 5e-2 * m and err.mean() <= 1e-2 * m, (err.max() / m, err.mean() / m)
    assert s.lens.tolist() == [150, 150, 0]


def test_sampling_and_graph_replay(cuda_dev, weights):
    """A captured step fed by its own sampled tokens equals eager steps, and the tokens follow the given uniforms."""
    u = torch.rand(12, 4, generator=torch.Generator().manual_seed(4)).to(cuda_dev)

    def fresh():
        s = BatchDecodeStep(weights, 4, 16, page=8, max_pages=4)
        s.active.fill_(1)
        s.tok.copy_(torch.tensor([5, 6, 7, 8]))
        s.temperature.copy_(torch.tensor([0.0, 0.7, 1.0, 1.0]))
        s.top_k.copy_(torch.tensor([0, 20, 0, 0]))
        s.top_p.copy_(torch.tensor([1.0, 0.9, 0.8, 1.0]))
        return s

    a, b = fresh(), fresh().capture()
    seen = []
    for row in u:
        for s, run in ((a, a.step), (b, b.replay)):
            s.u.copy_(row)
            run()
        assert torch.equal(a.tok, b.tok) and torch.equal(a.logits, b.logits) and torch.equal(a.lens, b.lens)
        assert int(a.tok[0]) == int(a.logits[0].float().argmax())
        seen.append(a.tok.tolist())
    assert len({tuple(t) for t in seen}) > 1
    assert torch.equal(a.table, b.table) and all(torch.equal(a.kc[i], b.kc[i]) for i in a.kc)


def test_every_norm_once(cuda_dev, weights):
    """The first norm comes with the embedding: quantizing its rows gives the codes of norm and quantization in one, and
    the step asks for the others, two a layer, only."""
    s = BatchDecodeStep(weights, 3, 4, page=16, max_pages=2)
    g = torch.Generator().manual_seed(6)
    s.tok.copy_(torch.randint(0, CFG.vocab, (3,), generator=g))
    s.active.fill_(1)
    calls = []

    class Spy:
        def __getattr__(self, name, inner=s.E):
            calls.append(name)
            return getattr(inner, name)

    s.E = Spy()
    s.step()
    assert calls.count("add_rmsnorm_q") == 2 * CFG.layers
    e = dict(device=cuda_dev)
    h, x = torch.empty(3, CFG.hidden, dtype=torch.bfloat16, **e), torch.empty(3, CFG.hidden, dtype=torch.bfloat16, **e)
    tok = torch.randint(0, CFG.vocab, (3,), generator=g).to(cuda_dev)
    a, b = [(torch.empty(3, CFG.hidden, dtype=torch.int8, **e), torch.empty(3, **e)) for _ in range(2)]
    s.K.embed_rmsnorm(tok, weights.embed, weights.norm[0], h, x, CFG.eps)
    s.E.quant_rows(x, *a)
    s.E.add_rmsnorm_q(h, None, weights.norm[0], *b, CFG.eps)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
