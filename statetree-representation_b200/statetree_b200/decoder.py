"""A minimal Qwen3-architecture decoder over the tree-stored layers, for decode-throughput measurement with random
weights: RMSNorm, fused q/k/v and gate/up projections, per-head q/k RMSNorm, RoPE, grouped-query attention over the
compressed KV pages, SwiGLU, untied lm_head, greedy sampling.  One decode step is captured in a CUDA graph and
replayed (the measurement method of the reference's statetree/bench.py:74-133 DecodeRunner).  `compressed=False`
builds the BF16 control from the same seeds: dense weights, a dense BF16 KV cache and FlashAttention.

Tensor parallelism (one process per GPU): q/k/v and gate/up are split by rows (heads / intermediate columns), o and
down by input columns with an all-reduce of their outputs, the lm_head by vocabulary rows with an all-gather of the
logits; embeddings and norms are replicated.  With `experts > 0` the MLP is a routed expert block (softmax router,
top-k, renormalised weights, TreeExperts): under several ranks the attention stays tensor-parallel and the experts are
split over the ranks (expert parallelism: every rank routes all tokens, computes its own experts' weighted partial
output, and the partial outputs are all-reduced).  Every rank draws the full tensors from the same seeds and keeps its slice,
so a tensor-parallel run computes the same function as the single-GPU one.

`eight_bit_kv=True` keeps the KV cache in 8-bit pages (kvcache.PageStore8) instead of the lossless ones: a decode step then norms,
rotates and appends through their append, and a prompt runs in one pass (prefill) over their chunk attention.

`whole_prompts=True` runs prompts in one pass over the lossless pages too: q/k/v rows are normed and rotated (rotary.rotate), appended, and
the queries attend to the pages (PageStore.chunk_attention); the o and down projections add the residual stream in their epilogue, and
SwiGLU is the gate/up projection's (TreeLinear.fused).  Probabilities of that attention are rounded to BF16, 2^-8 of each at most; decode
steps, which keep some sixteen bits of them, stay as they are.
"""
import math
from dataclasses import dataclass

import torch
import torch.distributed as dist
import torch.nn.functional as Fn

from .kvcache import PagedKVCache, decode_splits8
from .linear import TreeLinear, interleave_gate_up
from .ops import ext, kv_ext
from .rotary import rotate


def _flash():
    from flash_attn import flash_attn_with_kvcache
    return flash_attn_with_kvcache


@dataclass
class DecoderConfig:
    layers: int = 36
    hidden: int = 4096
    heads: int = 32
    kv_heads: int = 8
    head_dim: int = 128
    inter: int = 12288
    vocab: int = 151936
    rope_theta: float = 1e6
    eps: float = 1e-6
    experts: int = 0                 # > 0: the MLP of every layer is a routed mixture of experts (Qwen3-MoE shape)
    top_k: int = 8
    moe_inter: int = 768             # intermediate size of one expert
    distinct_experts: int = 4        # random expert matrices drawn per layer; the others are copies in their own buffers


class _Dense:
    """BF16 control for a TreeLinear: same call, dense weight"""

    def __init__(self, W):
        self.W = W
        self.out_features, self.in_features = W.shape

    def __call__(self, x):
        return Fn.linear(x, self.W)

    def record_bytes(self):
        return self.W.numel() * 2


class TreeDecoder:
    def __init__(self, cfg, device, batch, max_len, compressed=True, seed=0, rank=0, world=1, group=None,
                 eight_bit_kv=False, whole_prompts=False):
        self.cfg, self.dev, self.B, self.rank, self.world, self.group = cfg, torch.device(device), batch, rank, world, group
        self.compressed, self.eight_bit_kv = compressed, eight_bit_kv
        self.whole_prompts = eight_bit_kv or whole_prompts
        c = cfg
        assert compressed or not self.whole_prompts, "the BF16 control keeps its own cache"
        assert not whole_prompts or eight_bit_kv or c.head_dim == 128, "the lossless pages hold heads of dimension 128"
        assert c.heads % world == 0 and c.kv_heads % world == 0 and c.inter % (64 * world) == 0 and c.vocab % (16 * world) == 0
        self.hq, self.hkv = c.heads // world, c.kv_heads // world
        self.fused_act = False
        if c.experts:
            assert compressed, "the mixture-of-experts decoder has no BF16 control"
            assert c.experts % world == 0
            from .parallel import expert_partition
            self.e_lo, self.e_hi, self.emap = expert_partition(c.experts, rank, world, self.dev)
        if compressed and not c.experts and batch <= 8:
            from .ops import lib
            with torch.cuda.device(self.dev):
                self.fused_act = bool(lib().st_gemv_swiglu_supported(2 * c.inter // world, c.hidden, batch))
        gen = torch.Generator(device=self.dev)
        self._tid = 0

        def draw(rows, cols):
            gen.manual_seed(seed * 100003 + self._tid)
            self._tid += 1
            return (torch.randn(rows, cols, device=self.dev, generator=gen) * 0.02).to(torch.bfloat16)

        def make(W):
            return TreeLinear.from_weight(W.contiguous(), verify=False) if compressed else _Dense(W.contiguous())

        def rows(W, n_parts=1):
            per = W.shape[0] // world
            return W[rank * per:(rank + 1) * per]

        D = c.head_dim
        self.embed = make(draw(c.vocab, c.hidden))
        self.blocks = []
        for _ in range(c.layers):
            q, k, v = draw(c.heads * D, c.hidden), draw(c.kv_heads * D, c.hidden), draw(c.kv_heads * D, c.hidden)
            qkv = make(torch.cat([rows(q), rows(k), rows(v)]))
            del q, k, v
            o = draw(c.hidden, c.heads * D)
            per = o.shape[1] // world
            o = make(o[:, rank * per:(rank + 1) * per])
            if c.experts:
                gu, d = self._make_experts(draw), None
            else:
                g, u = draw(c.inter, c.hidden), draw(c.inter, c.hidden)
                if self.fused_act:                          # gate / up tiles in turn: SwiGLU in the GEMV's epilogue
                    gu = make(interleave_gate_up(rows(g).contiguous(), rows(u).contiguous()))
                else:
                    gu = make(torch.cat([rows(g), rows(u)]))
                del g, u
                d = draw(c.hidden, c.inter)
                per = d.shape[1] // world
                d = make(d[:, rank * per:(rank + 1) * per])
            self.blocks.append((qkv, o, gu, d))
        self.lm_head = make(rows(draw(c.vocab, c.hidden)))
        ones = torch.ones(c.hidden, dtype=torch.bfloat16, device=self.dev)
        self.norm_w, self.head_norm_w = ones, torch.ones(D, dtype=torch.bfloat16, device=self.dev)
        # rotary tables
        inv = 1.0 / (c.rope_theta ** (torch.arange(0, D, 2, device=self.dev, dtype=torch.float32) / D))
        ang = torch.arange(max_len, device=self.dev, dtype=torch.float32)[:, None] * inv[None]
        self.cos, self.sin = ang.cos().contiguous(), ang.sin().contiguous()      # float32 [max_len, 64]
        self.max_len = max_len
        self.pos_buf = torch.zeros(1, dtype=torch.long, device=self.dev)
        self.h_buf = torch.empty(batch, c.hidden, dtype=torch.bfloat16, device=self.dev)
        self.q_buf = torch.empty(batch, self.hq, D, dtype=torch.bfloat16, device=self.dev)
        self.k_buf = torch.empty(batch, self.hkv, D, dtype=torch.bfloat16, device=self.dev)
        self.tokens = torch.zeros(batch, dtype=torch.long, device=self.dev)
        if compressed:
            self.cache = PagedKVCache(c.layers, batch, max_len, self.hkv, self.dev, pool_blocks=1 << 14, eight_bit=eight_bit_kv,
                                      head_dim=D)
        else:
            self.kc = [torch.zeros(batch, max_len, self.hkv, D, dtype=torch.bfloat16, device=self.dev) for _ in range(c.layers)]
            self.vc = [torch.zeros_like(k) for k in self.kc]
            self.lens = torch.zeros(batch, dtype=torch.int32, device=self.dev)
        self.comm = None
        if world > 1 and batch <= 64 and c.hidden <= 8192 and c.hidden % 8 == 0:
            from .parallel import peer_comm
            self.comm = peer_comm(group)
        self.graph = None
        # RMSNorm(x + delta) formed inside the GEMV that consumes it (no add + norm launch in front of q/k/v, gate/up
        # and the output head) where the kernel takes the shape
        self.pre_qkv = self.pre_gu = self.pre_head = False
        if compressed and batch <= 8:
            E = ext()
            qkv0, _, gu0, _ = self.blocks[0]
            with torch.cuda.device(self.dev):
                self.pre_qkv = E.gemv_prenorm_supported(qkv0.out_features, c.hidden, batch, False)
                self.pre_gu = (not c.experts) and E.gemv_prenorm_supported(gu0.out_features, c.hidden, batch, self.fused_act)
                self.pre_head = E.gemv_prenorm_supported(self.lm_head.out_features, c.hidden, batch, False)
            self._xbuf = [torch.empty(batch, c.hidden, dtype=torch.bfloat16, device=self.dev) for _ in range(2)]

    def _prenorm_linear(self, layer, x, delta, act=False):
        """(layer(RMSNorm(x + delta) * w), x + delta) in one launch; the new residual stream goes to the buffer x is not in"""
        from .linear import _state
        E = ext()
        B, M, N = x.shape[0], layer.out_features, layer.in_features
        eo, el, eb = layer.tables()
        y = torch.empty(B, M // 2 if act else M, dtype=torch.bfloat16, device=self.dev)
        x_out = None
        if delta is not None:
            x_out = self._xbuf[1] if x is self._xbuf[0] else self._xbuf[0]
        ws = _state(self.dev).get_ws(E.gemv_workspace_bytes(M, N, B))
        E.gemv_prenorm(layer.tree, eo, eb, el, x, delta, self.norm_w, self.cfg.eps, x_out, y, ws, act)
        return y, (x if x_out is None else x_out)

    def _make_experts(self, draw):
        """(router weight [E, hidden] BF16, TreeExperts over this rank's experts): `distinct_experts` random matrices per
        projection, every expert a copy of one of them in a buffer of its own (so the records of every expert a step
        touches stream from HBM), which keeps building a 128-expert x 48-layer model within minutes"""
        from .experts import TreeExperts
        c = self.cfg
        router = draw(c.experts, c.hidden)
        base13 = [TreeLinear.from_weight(draw(2 * c.moe_inter, c.hidden), verify=False) for _ in range(c.distinct_experts)]
        base2 = [TreeLinear.from_weight(draw(c.hidden, c.moe_inter), verify=False) for _ in range(c.distinct_experts)]

        def copy_of(tl):
            m = TreeLinear(tl.in_features, tl.out_features, device="meta", n_esc=tl.esc_rows.numel())
            m._buffers["tree"] = tl.tree.clone()
            for k in ("esc_rows", "esc_cols", "esc_bits"):
                m._buffers[k] = tl._buffers[k]
            m._tables = tl.tables()
            return m

        mine = range(self.e_lo, self.e_hi)
        te = TreeExperts([copy_of(base13[e % c.distinct_experts]) for e in mine],
                         [copy_of(base2[e % c.distinct_experts]) for e in mine])
        te.tables()
        return (router, te)

    def weight_bytes(self):
        """record bytes a decode step reads on this rank (the embedding table is read B rows at a time; of the experts,
        an upper bound: min(experts on the rank, batch x top_k) of them)"""
        n = self.lm_head.record_bytes()
        for qkv, o, gu, d in self.blocks:
            n += qkv.record_bytes() + o.record_bytes()
            if self.cfg.experts:
                te = gu[1]
                per = te.record_bytes() // te.num_experts
                n += per * min(te.num_experts, self.B * self.cfg.top_k)
            else:
                n += gu.record_bytes() + d.record_bytes()
        return n

    def _row_parallel(self, layer, xin):
        """(delta, summed): the output of a row-parallel projection (o, down) on this rank's activation slice.  A tree
        layer at GEMV batch sizes sums over the ranks inside its own kernel (summed = True); otherwise the partial
        output comes back and _add_norm adds the ranks."""
        from .linear import GEMV_AR_MAX, GEMV_MAX, _state
        B = xin.shape[0]
        if (self.world > 1 and self.comm is not None and self.compressed and B <= min(GEMV_MAX, GEMV_AR_MAX)
                and layer.bias is None and self.comm.gemv_allreduce_fits(layer.out_features, B)):
            eo, el, eb = layer.tables()
            y = torch.empty(B, layer.out_features, dtype=torch.bfloat16, device=self.dev)
            ws = _state(self.dev).get_ws(ext().gemv_workspace_bytes(layer.out_features, layer.in_features, B))
            self.comm.gemv_allreduce(layer.tree, eo, eb, el, xin, y, ws)
            return y, True
        return layer(xin), False

    def _add_norm(self, x, delta, h, summed=False):
        """x += (all-reduced) delta; h = RMSNorm(x) * w.  Under tensor parallelism delta is this rank's partial output of
        a row-parallel projection unless `summed`: one kernel sums it over the ranks through peer memory and applies
        add + norm."""
        c = self.cfg
        if delta is not None and self.world > 1 and not summed:
            if self.comm is not None:
                self.comm.all_reduce_add_rmsnorm(x, delta, self.norm_w, h, c.eps)
                return
            dist.all_reduce(delta, group=self.group)
        ext().add_rmsnorm(x, delta, self.norm_w, h, c.eps)

    def _append8(self, layer, qkv, slots, positions, q_out):
        """fused q/k/v rows [N, (hq + 2 hkv) D] into an 8-bit layer's pages, normed and rotated queries into q_out; the layer"""
        q, k, v = qkv.view(qkv.shape[0], self.hq + 2 * self.hkv, self.cfg.head_dim).split([self.hq, self.hkv, self.hkv], 1)
        layer.append(k, v, slots, positions, self.cos, self.sin, True, q, self.head_norm_w, self.head_norm_w, self.cfg.eps, q_out)
        return layer

    def prefill(self, prompt):
        """prompt [B, P] token ids behind whatever the cache holds, in one pass: every layer's keys and values go into the pages,
        then its queries attend to them (causal).  Returns the logits of every sequence's last token [B, vocab]"""
        if not self.whole_prompts or self.world > 1:
            raise RuntimeError("TreeDecoder.prefill: a single-GPU decoder with eight_bit_kv=True or whole_prompts=True")
        c, E, (B, P) = self.cfg, ext(), prompt.shape
        if B != self.B:
            raise ValueError(f"TreeDecoder.prefill: {B} sequences, the decoder was made for {self.B}")
        if not P:
            raise ValueError("TreeDecoder.prefill: no tokens")
        start = int(self.pos_buf.item())
        if start + P > self.max_len:
            raise ValueError(f"TreeDecoder.prefill: {P} tokens from position {start} exceed the cache capacity of {self.max_len} tokens")
        N, D, cache = B * P, c.head_dim, self.cache
        cache._stored = start                                # (decode steps count on the GPU only)
        slots = cache.begin_chunk(B, P)
        positions = (start + torch.arange(P, device=self.dev)).repeat(B)
        cu = torch.arange(0, N + 1, P, dtype=torch.int32, device=self.dev)
        x = self.embed.rows(prompt.reshape(-1))
        h = torch.empty(N, c.hidden, dtype=torch.bfloat16, device=self.dev)
        q = torch.empty(N, self.hq, D, dtype=torch.bfloat16, device=self.dev)
        delta = None
        for li, (qkv, o, gu, d) in enumerate(self.blocks):
            if not self.eight_bit_kv:
                delta = self._prefill_block(li, x, delta, h, slots, positions, cu)
                continue
            E.add_rmsnorm(x, delta, self.norm_w, h, c.eps)
            layer = self._append8(cache.layers[li], qkv(h), slots, positions, q)
            att = layer.chunk_attention(q, cu, cache.bt32[:B], cache.lens[:B], 1.0 / math.sqrt(D))
            E.add_rmsnorm(x, o(att.view(N, self.hq * D)), self.norm_w, h, c.eps)
            if c.experts:
                router, te = gu
                delta = te(h, *E.moe_route(Fn.linear(h, router), c.top_k, True, None), None)
                continue
            y = gu(h)
            if self.fused_act:                               # (16-row tiles of gate and up in turn)
                y = y.view(N, c.inter // 16, 2, 16).transpose(1, 2).reshape(N, 2 * c.inter)
            act = torch.empty(N, c.inter, dtype=torch.bfloat16, device=self.dev)
            E.silu_mul(y, act)
            delta = d(act)
        last = torch.arange(P - 1, N, P, device=self.dev)
        E.add_rmsnorm(x, delta, self.norm_w, h, c.eps)
        cache.end_chunk(P)
        self.pos_buf += P
        return self.lm_head(h[last])

    def _prefill_block(self, li, x, delta, h, slots, positions, cu):
        """layer li of a prompt pass over the lossless pages: x (the residual stream, after the experts' `delta` of the layer before, if
        any) is added to in place; returns this layer's experts' output, which the next norm adds, or None"""
        c, E, (N, D), layer = self.cfg, ext(), (x.shape[0], self.cfg.head_dim), self.cache.layers[li]
        qkv, o, gu, d = self.blocks[li]
        E.add_rmsnorm(x, delta, self.norm_w, h, c.eps)
        q, k, v = qkv.fused(h).view(N, self.hq + 2 * self.hkv, D).split([self.hq, self.hkv, self.hkv], 1)
        q, k = rotate(q, k, positions, self.cos, self.sin, q_norm=self.head_norm_w, k_norm=self.head_norm_w, eps=c.eps)
        layer.append(k, v, slots)
        att = layer.chunk_attention(q, cu, self.cache.bt32[:self.B], self.cache.lens[:self.B], 1.0 / math.sqrt(D))
        o.fused(att.view(N, self.hq * D), residual=x, out=x)
        E.add_rmsnorm(x, None, self.norm_w, h, c.eps)
        if c.experts:
            router, te = gu
            return te(h, *E.moe_route(Fn.linear(h, router), c.top_k, True, None), None)
        if self.fused_act:                                   # (16-row tiles of gate and up in turn)
            act = gu.fused(h, "swiglu")
        else:
            act = torch.empty(N, c.inter, dtype=torch.bfloat16, device=self.dev)
            E.silu_mul(gu.fused(h), act)
        d.fused(act, residual=x, out=x)
        return None

    def _step(self):
        """one decode step for self.tokens at position self.pos; about ten launches per layer"""
        c, B, D = self.cfg, self.B, self.cfg.head_dim
        E = ext()
        x = self.embed.rows(self.tokens) if self.compressed else self.embed.W[self.tokens]
        scale = 1.0 / math.sqrt(D)
        h, qb, kb = self.h_buf, self.q_buf, self.k_buf
        slots = self.cache.begin_step(B) if self.compressed else None
        delta, summed = None, False
        for li, (qkv, o, gu, d) in enumerate(self.blocks):
            if self.pre_qkv and (delta is None or summed or self.world == 1):
                y, x = self._prenorm_linear(qkv, x, delta)
            else:
                self._add_norm(x, delta, h, summed)
                y = qkv(h)
            if self.eight_bit_kv:                           # norm + rope of q and k and the append of k, v: one launch
                att = self._append8(self.cache.layers[li], y, slots, self.pos_buf, qb).attention(
                    qb, self.cache.bt32[:B], self.cache.lens[:B], scale, self.splits, None, 4)
            elif self.compressed:
                layer = self.cache.layers[li]
                kv_ext().rope_append(y, self.head_norm_w, self.head_norm_w, self.cos, self.sin, self.pos_buf, qb,
                                     self.hq, self.hkv, c.eps, slots, layer.pages, layer.pool, layer.pcnt)
                att = layer.attention(qb, self.cache.bt32[:B], self.cache.lens[:B], scale, self.splits, None, 4)
            else:
                E.qk_norm_rope(y, self.head_norm_w, self.head_norm_w, self.cos, self.sin, self.pos_buf, qb, kb, c.eps)
                v = y[:, (self.hq + self.hkv) * D:].view(B, self.hkv, D)
                att = _flash()(qb.view(B, 1, self.hq, D), self.kc[li], self.vc[li], k=kb.view(B, 1, self.hkv, D),
                               v=v.unsqueeze(1), cache_seqlens=self.lens, softmax_scale=scale)
            delta, summed = self._row_parallel(o, att.reshape(B, self.hq * D))
            if self.pre_gu and (summed or self.world == 1):
                act, x = self._prenorm_linear(gu, x, delta, self.fused_act)
                if not self.fused_act:
                    y2 = act
                    act = torch.empty(B, y2.shape[1] // 2, dtype=torch.bfloat16, device=self.dev)
                    E.silu_mul(y2, act)
                delta, summed = self._row_parallel(d, act)
                continue
            self._add_norm(x, delta, h, summed)
            if c.experts:
                router, te = gu
                # softmax, top-k and renormalisation in one launch; with few pairs under expert parallelism the router
                # also maps the ids to this rank's experts (foreign pairs: weight 0), which the experts then run as is
                from .experts import SLOT_MAX
                logits = Fn.linear(h, router)
                if self.world > 1 and B * c.top_k <= SLOT_MAX:
                    ids, w = E.moe_route(logits, c.top_k, True, self.emap)
                    delta, summed = te(h, ids, w, None), False
                else:
                    ids, w = E.moe_route(logits, c.top_k, True, None)
                    delta, summed = te(h, ids, w, self.emap if self.world > 1 else None), False
                continue                                     # (the all-reduce over ranks happens in the next _add_norm)
            if self.fused_act:
                act = gu.swiglu(h)
            else:
                y = gu(h)
                act = torch.empty(B, y.shape[1] // 2, dtype=torch.bfloat16, device=self.dev)
                E.silu_mul(y, act)
            delta, summed = self._row_parallel(d, act)
        if self.pre_head and (summed or self.world == 1):
            logits, x = self._prenorm_linear(self.lm_head, x, delta)
        else:
            self._add_norm(x, delta, h, summed)
            logits = self.lm_head(h)
        if self.world > 1:
            parts = [torch.empty_like(logits) for _ in range(self.world)]
            dist.all_gather(parts, logits, group=self.group)
            logits = torch.cat(parts, 1)
        if self.compressed:
            self.cache.end_step()
        else:
            self.lens += 1
        self.pos_buf += 1
        return logits

    def _pick(self, logits):
        """greedy: next_tok = argmax of every row"""
        if self.compressed and logits.is_contiguous() and logits.shape[1] % 8 == 0 and logits.data_ptr() % 16 == 0:
            ext().argmax(logits, self.next_tok)
        else:
            self.next_tok.copy_(logits.argmax(-1))

    def capture(self):
        from .kvcache import decode_splits
        pages = (self.max_len + 15) // 16
        self.splits = (decode_splits8(self.B * self.hkv * -(-self.hq // (8 * self.hkv)), pages) if self.eight_bit_kv else
                       decode_splits(self.B, self.hkv, pages) if self.compressed else 1)
        self.next_tok = torch.zeros(self.B, dtype=torch.long, device=self.dev)
        side = torch.cuda.Stream(self.dev)
        side.wait_stream(torch.cuda.current_stream(self.dev))      # weights and buffers were written on that stream
        with torch.cuda.stream(side):
            for _ in range(2):                                   # warm-up steps (also sizes every workspace)
                self._pick(self._step())
        side.synchronize()
        self.reset()
        torch.cuda.synchronize(self.dev)
        self.graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(self.graph, stream=side):
            logits = self._step()
            self._pick(logits)
        self.logits = logits
        self.reset()
        torch.cuda.synchronize(self.dev)
        self._check_status("capture")

    def _check_status(self, where):
        """a kernel that gave up on a bounded wait (a peer that never arrived) leaves its output unwritten: fail loudly"""
        from .ops import device_status
        with torch.cuda.device(self.dev):
            code = device_status()
        if code != 0:
            raise RuntimeError(f"TreeDecoder.{where}: a kernel gave up on a bounded wait (device status {code}); the "
                               "results of this call are invalid")

    def reset(self):
        self.pos_buf.zero_()
        if self.compressed:
            self.cache.reset()
        else:
            self.lens.zero_()

    def run(self, prompt, n_new, collect=None, margins=None):
        """prompt [B, P] token ids (teacher-forced one step at a time; with an 8-bit cache or whole_prompts in one pass), then n_new greedy tokens ->
        [B, n_new].
        collect (optional list): receives the model's prediction after every prompt step (teacher-forced top-1).
        margins (optional list): receives, per generated token, the top-2 logit margin of sequence 0 that chose it."""
        start = int(self.pos_buf.item())
        if start + prompt.shape[1] + n_new > self.max_len:       # beyond it the page lookup would leave the block table
            raise ValueError(f"TreeDecoder.run: {prompt.shape[1]} prompt + {n_new} new tokens from position {start} "
                             f"exceed the cache capacity of {self.max_len} tokens")
        out = []
        whole = self.whole_prompts and self.world == 1 and collect is None and prompt.shape[1] > 1
        if whole:
            self.logits.copy_(self.prefill(prompt))
            self._pick(self.logits)
        for t in range(0 if not whole else prompt.shape[1], prompt.shape[1]):
            self.tokens.copy_(prompt[:, t])
            self.graph.replay()
            if collect is not None:
                collect.append(self.next_tok.clone())
        for _ in range(n_new):
            if margins is not None:
                top2 = self.logits[0].float().topk(2).values
                margins.append(top2[0] - top2[1])
            self.tokens.copy_(self.next_tok)
            out.append(self.next_tok.clone())
            self.graph.replay()
        res = torch.stack(out, 1) if out else torch.empty(self.B, 0, dtype=torch.long, device=self.dev)
        if self.world > 1:
            self._check_status("run")
        return res
