"""Prompts in one pass over the lossless pages where models use them: the decode runner (projections with epilogues, rotation, append, chunk
attention one behind the other) against a 64-bit forward pass, the Hugging Face cache with paged_prompts against a cache-free model, and
the vLLM data path."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _forward(m, tokens):
    """logits float64 [T, vocab] of one sequence: the runner's function without its BF16 roundings"""
    c, D, T = m.cfg, m.cfg.head_dim, len(tokens)
    W = lambda layer: layer.dequantize().double()                                       # noqa: E731
    norm = lambda y: y / (y.square().mean(-1, keepdim=True) + c.eps).sqrt()             # noqa: E731
    x = W(m.embed)[torch.tensor(tokens, device="cuda")]
    cos, sin = m.cos[:T, None].double(), m.sin[:T, None].double()

    def rot(y):
        a, b = y[..., 0::2], y[..., 1::2]
        return torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    hide = torch.ones(T, T, dtype=torch.bool, device="cuda").triu(1)
    for qkv, o, gu, d in m.blocks:
        q, k, v = (norm(x) @ W(qkv).t()).view(T, -1, D).split([m.hq, m.hkv, m.hkv], 1)
        q, k = rot(norm(q)), rot(norm(k))
        k, v = (t.repeat_interleave(m.hq // m.hkv, 1) for t in (k, v))
        p = torch.softmax((torch.einsum("ihd,jhd->hij", q, k) / math.sqrt(D)).masked_fill(hide, -math.inf), -1)
        x = x + torch.einsum("hij,jhd->ihd", p, v).flatten(1) @ W(o).t()
        g = W(gu)
        if m.fused_act:
            g = g.view(c.inter // 16, 2, 16, c.hidden).transpose(0, 1).reshape(2 * c.inter, c.hidden)
        g, u = (norm(x) @ g.t()).chunk(2, -1)
        x = x + (torch.nn.functional.silu(g) * u) @ W(d).t()
    return norm(x) @ W(m.lm_head).t()


# Two layers of about ten roundings to BF16 (2^-8 each) on the way of a value: 20 * 2^-8 at most
REL = 20 * 2.0 ** -8


@pytest.mark.parametrize("batch,P", [(1, 21), (3, 21), (2, 150), (9, 40)])
def test_decoder_prompts(batch, P):
    """in one pass, in two chunks, step by step: the same logits and pages up to roundings, all near 64 bits.  Nine sequences: gate and up
    are not interleaved"""
    from statetree_b200 import ops
    from statetree_b200.decoder import DecoderConfig, TreeDecoder
    cfg = DecoderConfig(layers=2, hidden=512, heads=4, kv_heads=2, head_dim=128, inter=1024, vocab=2048)
    new = 5
    m = TreeDecoder(cfg, "cuda", batch, P + new + 8, seed=5, whole_prompts=True)
    prompt = torch.randint(0, cfg.vocab, (batch, P), generator=torch.Generator().manual_seed(2)).cuda()
    want = [_forward(m, prompt[b].tolist()) for b in range(batch)]
    m.capture()
    for t in range(P):
        m.tokens.copy_(prompt[:, t])
        m.graph.replay()
    steps, by_step = m.logits.double(), [layer.dense() for layer in m.cache.layers]
    m.reset()
    one = m.prefill(prompt).double()
    at_once = [layer.dense() for layer in m.cache.layers]
    m.reset()
    cut = P * 2 // 3
    first, second = m.prefill(prompt[:, :cut]).double(), m.prefill(prompt[:, cut:]).double()
    m.cache.check()
    rel = lambda a, b: float((a - b).norm() / b.norm())                                       # noqa: E731
    for b in range(batch):
        assert rel(one[b], want[b][-1]) < REL and rel(second[b], want[b][-1]) < REL and rel(first[b], want[b][cut - 1]) < REL
        assert rel(steps[b], want[b][-1]) < REL
    for whole in (at_once, [layer.dense() for layer in m.cache.layers]):
        for (k0, v0), (k1, v1) in zip(by_step, whole):
            assert rel(k1.double(), k0.double()) < REL and rel(v1.double(), v0.double()) < REL
    runs = []
    for _ in range(2):                                       # the prompt in one pass, then steps from the graph
        m.reset()
        runs.append(m.run(prompt, new))
        assert int(m.cache.cum) == P + new == int(m.pos_buf)
    assert torch.equal(runs[0], runs[1])
    with pytest.raises(ValueError, match="capacity"):
        m.prefill(prompt)
    with pytest.raises(ValueError, match="sequences"):
        m.prefill(prompt[:1].expand(batch + 1, P))
    with pytest.raises(ValueError, match="no tokens"):
        m.prefill(prompt[:, :0])
    assert ops.device_status() == 0


def test_decoder_with_experts():
    from statetree_b200.decoder import DecoderConfig, TreeDecoder
    cfg = DecoderConfig(layers=2, hidden=512, heads=4, kv_heads=1, head_dim=128, vocab=1024, experts=8, top_k=2, moe_inter=256)
    m = TreeDecoder(cfg, "cuda", 2, 64, seed=1, whole_prompts=True)
    m.capture()
    prompt = torch.randint(0, cfg.vocab, (2, 33), generator=torch.Generator().manual_seed(3)).cuda()
    for t in range(33):
        m.tokens.copy_(prompt[:, t])
        m.graph.replay()
    steps = m.logits.double()
    m.reset()
    whole = m.prefill(prompt).double()
    assert float((whole - steps).norm() / steps.norm()) < 2 * REL      # (both with the roundings above)


@pytest.mark.parametrize("windows", [None, ["sliding_attention", "full_attention"], ["full_attention", "sliding_attention"]])
@pytest.mark.parametrize("pad", [0, 5, 19])
def test_hf_cache(windows, pad):
    """a prompt in two chunks (longer than the windows; padding beyond the first) and decode steps against a cache-free pass"""
    pytest.importorskip("transformers")
    from transformers import Qwen3Config, Qwen3ForCausalLM
    from statetree_b200.kvcache import StateTreeKVCache, enable
    cfg = Qwen3Config(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=128, max_position_embeddings=256, tie_word_embeddings=False,
                      **(dict(use_sliding_window=True, sliding_window=8, layer_types=windows) if windows else {}))
    torch.manual_seed(0)
    model = Qwen3ForCausalLM(cfg).to(torch.bfloat16).cuda().eval()
    B, P, steps = 2, 29, 6
    ids = torch.randint(0, cfg.vocab_size, (B, P + steps), device="cuda")
    mask = torch.ones(B, P + steps, dtype=torch.long, device="cuda")
    mask[1, :pad] = 0
    with torch.no_grad():
        full = model(input_ids=ids, attention_mask=mask).logits.float()
        enable(model)
        cache = StateTreeKVCache(model.config, batch_size=B, max_cache_len=P + steps + 8, paged_prompts=True)
        for _ in range(2):                                   # (and again after a reset)
            got = []
            for a, b in [(0, 17), (17, P)] + [(P + t, P + t + 1) for t in range(steps - 1)]:
                out = model(input_ids=ids[:, a:b], attention_mask=mask[:, :b], past_key_values=cache, use_cache=True)
                got.append((b, out.logits[:, -1].float()))
            cache.check()
            for n, g in got:
                want = full[:, n - 1]
                live = [b for b in range(B) if n - 1 >= (pad if b else 0)]
                assert float((g - want)[live].norm() / want[live].norm()) < 3e-2, n            # BF16 model: roundings fall differently
            cache.reset()


def test_hf_cache_refuses_other_masks():
    """packed sequences: a block-diagonal mask"""
    pytest.importorskip("transformers")
    import types
    from statetree_b200.kvcache import StateTreeKVCache, statetree_attention
    cfg = types.SimpleNamespace(num_hidden_layers=1, num_attention_heads=2, num_key_value_heads=2)
    cache = StateTreeKVCache(cfg, batch_size=1, max_cache_len=64, paged_prompts=True)
    k = torch.zeros(1, 2, 8, 128, dtype=torch.bfloat16, device="cuda")
    keys, values = cache.layers[0].update(k, k)
    odd = torch.ones(8, 8, dtype=torch.bool, device="cuda").tril()
    odd[4:, :4] = False
    with pytest.raises(ValueError, match="mask"):
        statetree_attention(types.SimpleNamespace(layer_idx=0, is_causal=True), k, keys, values, odd[None, None])
    cache.reset()
    keys, values = cache.layers[0].update(k, k)
    with pytest.raises(ValueError, match="softcap"):
        statetree_attention(types.SimpleNamespace(layer_idx=0, is_causal=True), k, keys, values, None, softcap=30.0)


def test_vllm_prefill():
    """PageBackend.prefill: chunks behind cached context and single tokens in one call, padded rows left alone"""
    from statetree_b200.vllm_kv import PageBackend, SharedPool
    HQ, H, D, nb = 8, 2, 128, 64
    sh = SharedPool("cuda", HQ, H, pool_mb=2)
    be = PageBackend(HQ, H, 1.0 / math.sqrt(D), sh)
    cache = torch.zeros(nb, H, 16, 400, dtype=torch.uint8, device="cuda")
    g = torch.Generator("cuda").manual_seed(0)
    ctx, new = [150, 40, 77], [60, 40, 1]
    bt = torch.randperm(nb, device="cuda", generator=g)[:60].to(torch.int32).view(3, 20)
    K, V = ([torch.randn(n, H, D, device="cuda", generator=g).to(torch.bfloat16) for n in ctx] for _ in range(2))
    for b, n in enumerate(ctx):
        pos = torch.arange(n, device="cuda")
        be.write(K[b].view(n, H * D), V[b].view(n, H * D), cache, bt[b].long()[pos // 16] * 16 + pos % 16)
    q = torch.randn(sum(new) + 3, HQ * D, device="cuda", generator=g).to(torch.bfloat16)
    cu = torch.tensor([0, 60, 100, 101], dtype=torch.int32, device="cuda")
    out = torch.full_like(q, 5.0)
    for window in (0, 30):
        be.prefill(q, cache, bt, cu, torch.tensor(ctx, dtype=torch.int32, device="cuda"), out, window=window)
        assert bool((out[101:] == 5).all())
        for b, (n, m) in enumerate(zip(ctx, new)):
            at, j = torch.arange(n - m, n, device="cuda")[:, None], torch.arange(n, device="cuda")[None]
            hide = (j > at) | ((j <= at - window) if window else j < 0)
            k, v = (t[b].double().repeat_interleave(HQ // H, 1) for t in (K, V))
            rows = q[int(cu[b]):int(cu[b + 1])].view(m, HQ, D).double()
            p = torch.softmax((torch.einsum("ihd,jhd->hij", rows, k) / math.sqrt(D)).masked_fill(hide, -math.inf), -1)
            want = torch.einsum("hij,jhd->ihd", p, v)
            got = out[int(cu[b]):int(cu[b + 1])].view(m, HQ, D).double()
            assert float((got - want).norm() / want.norm()) < 5e-3
