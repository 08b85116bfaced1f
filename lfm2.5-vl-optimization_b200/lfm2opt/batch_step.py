"""One LFM2 decode step for a batch of requests at different positions, over a paged KV cache, with sampling.

The batched sibling of decode_step.DecodeStep (batch 1, dense cache, argmax): the W8A8 linears (int8_ext) on the same
weights, and the four batched-serving operators in the order a serving loop runs them:

  kv_slots: a page and a slot for every active request's token
  embedding and first norm (embed_rmsnorm) -> per layer norm + quantization (add_rmsnorm_q), then either
    attention:  qkv GEMM -> qk_norm_rope_kv_paged (k, v into their slots) -> tree_attention (one query a request) -> o GEMM
    short conv: in_proj GEMM -> shortconv_step -> out_proj GEMM
  and w1|w3 GEMM with the SwiGLU -> w2 GEMM
  lm_head GEMM -> sample_next

A step runs on the device without a synchronisation, so it captures into a CUDA graph (`capture`). A request that is not
active, for which there is no free page, or that holds max_pages full pages, sits the step out: its token, length and
convolution states stay.
"""

import torch

from .kernels import ext, int8_ext

BF = torch.bfloat16


class BatchDecodeStep:
    """State and buffers of batched decode for `weights` (decode_step.Lfm2Weights).

    requests: request slots; num_pages: pages of the pool (each holds `page` positions of every attention layer);
    max_pages: pages of one request at most. Tensors a caller sets between steps: active int32 [requests] (1: decodes),
    tok int64 [requests] (the token to feed; replaced by the sampled one), temperature / top_p / min_p fp32 and top_k int32
    [requests], u fp32 [requests] (the step's uniforms). lens int32 [requests] are the cached positions."""

    def __init__(self, weights, requests, num_pages, page=64, max_pages=64):
        self.w, self.cfg, self.B, self.page = weights, weights.cfg, requests, page
        self.K, self.E = ext(), int8_ext()
        c, dev, B = self.cfg, weights.embed.device, requests
        H, NQ, NKV, D = c.hidden, c.n_heads, c.n_kv, c.head_dim

        def buf(*shape, dtype=BF):
            return torch.zeros(*shape, dtype=dtype, device=dev)

        i32 = dict(dtype=torch.int32, device=dev)
        self.kc = {i: buf(num_pages, NKV, page, D) for i in c.attn_layers}
        self.vc = {i: buf(num_pages, NKV, page, D) for i in c.attn_layers}
        self.conv = {i: buf(B, H, c.conv_len) for i in range(c.layers) if i not in c.attn_layers}
        self.table = torch.full((B, max_pages), -1, **i32)
        self.free, self.n_free = torch.arange(num_pages, **i32), torch.tensor([num_pages], **i32)
        self.lens, self.want, self.got, self.active = (torch.zeros(B, **i32) for _ in range(4))
        self.cu = torch.zeros(B + 1, **i32)
        self.rows = torch.arange(B + 1, **i32)  # tree_attention: one query a request
        self.positions, self.slots = buf(B, dtype=torch.long), buf(B, dtype=torch.long)
        self.tok, self.new_tok = buf(B, dtype=torch.long), buf(B, dtype=torch.long)
        self.temperature, self.top_p = torch.ones(B, device=dev), torch.ones(B, device=dev)
        self.min_p, self.u = torch.zeros(B, device=dev), torch.zeros(B, device=dev)
        self.top_k = torch.zeros(B, **i32)
        self.h, self.x, self.y = buf(B, H), buf(B, H), buf(B, H)
        self.qkv, self.q, self.o = buf(B, (NQ + 2 * NKV) * D), buf(B, NQ, D), buf(B, NQ, D)
        self.bcx, self.cy, self.act = buf(B, 3 * H), buf(B, H), buf(B, c.inter)
        self.hold = buf(B, H, c.conv_len)
        wide = max(H, c.inter, NQ * D)
        self.q8, self.s8 = buf(B * wide, dtype=torch.int8), buf(B, dtype=torch.float32)
        self.logits = buf(B, c.vocab)
        S = self.K.tree_attention_splits(B, NQ, NKV, D, 1, max_pages * page)
        self.ws = buf(B, NQ, S, D + 2, dtype=torch.float32) if S > 1 else None
        self.inv_freq = weights.inv_freq
        self.graph = None

    def _codes(self, k):
        return self.q8[:self.B * k].view(self.B, k)

    def _linear(self, x, wq, y):
        """y = x wq^T for bf16 x [B, K]: quantized per token, then the W8A8 GEMM."""
        codes = self._codes(x.shape[-1])
        self.E.quant_rows(x, codes, self.s8)
        self.E.gemm_i8(codes, self.s8, wq[0], wq[1], None, y, False)

    @torch.no_grad()
    def step(self):
        K, E, W, c, B = self.K, self.E, self.w, self.cfg, self.B
        torch.add(self.lens, self.active, out=self.want)
        K.kv_slots(self.lens, self.want, self.table, self.free, self.n_free, self.page, self.got, self.cu, self.positions,
                   self.slots)
        # rows of the step are requests; the granted tokens are packed
        runs = self.cu[1:] > self.cu[:-1]
        at = self.cu[:-1].long().clamp_(max=B - 1)
        pos, slot = self.positions[at], torch.where(runs, self.slots[at], -1)
        K.embed_rmsnorm(self.tok, W.embed, W.norm[0], self.h, self.x, c.eps)
        codes = self._codes(c.hidden)
        E.quant_rows(self.x, codes, self.s8)
        for i, L in enumerate(W.layer):
            if i in c.attn_layers:
                E.gemm_i8(codes, self.s8, L["qkv"][0], L["qkv"][1], None, self.qkv, False)
                K.qk_norm_rope_kv_paged(self.qkv, L["qw"], L["kw"], self.inv_freq, 1.0, pos, slot, self.q, self.kc[i],
                                        self.vc[i], c.eps)
                K.tree_attention(self.q, self.kc[i], self.vc[i], self.table, self.lens, self.rows, None, self.o, self.ws,
                                 c.head_dim ** -0.5, 1)
                self._linear(self.o.view(B, -1), L["o"], self.y)
            else:
                E.gemm_i8(codes, self.s8, L["in"][0], L["in"][1], None, self.bcx, False)
                self.hold.copy_(self.conv[i])
                K.shortconv_step(self.bcx, self.conv[i], L["cw"], None, self.cy)
                torch.where(runs[:, None, None], self.conv[i], self.hold, out=self.conv[i])
                self._linear(self.cy, L["out"], self.y)
            E.add_rmsnorm_q(self.h, self.y, W.ffn_norm[i], codes, self.s8, c.eps)
            E.gemm_i8_silu(codes, self.s8, L["w13"][0], L["w13"][1], None, self.act)
            self._linear(self.act, L["w2"], self.y)
            E.add_rmsnorm_q(self.h, self.y, W.norm[i + 1], codes, self.s8, c.eps)
        E.gemm_i8(codes, self.s8, W.head[0], W.head[1], None, self.logits, False)
        K.sample_next(self.logits, self.temperature, self.top_k, self.top_p, self.min_p, self.u, self.new_tok)
        torch.where(runs, self.new_tok, self.tok, out=self.tok)
        self.lens.copy_(self.got)

    @torch.no_grad()
    def release(self, request):
        """End a request: its pages go back to the pool, its slot is empty (length 0, convolution states zero)."""
        self.active[request] = 0
        want = self.lens.clone()
        want[request] = 0
        self.K.kv_slots(self.lens, want, self.table, self.free, self.n_free, self.page, self.got, self.cu,
                        self.positions, self.slots)
        self.lens.copy_(self.got)
        for st in self.conv.values():
            st[request] = 0

    def capture(self):
        """Capture a step into a CUDA graph (after one eager step on a side stream with no request active, which changes
        nothing). `replay()` then runs a step."""
        dev, active = self.h.device, self.active.clone()
        side = torch.cuda.Stream(dev)
        self.active.zero_()
        side.wait_stream(torch.cuda.current_stream(dev))
        with torch.cuda.stream(side):
            self.step()
        torch.cuda.current_stream(dev).wait_stream(side)
        self.active.copy_(active)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=side):  # (its own stream may be one of another device)
            self.step()
        return self

    def replay(self):
        self.graph.replay()
