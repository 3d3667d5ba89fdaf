"""The 8-bit KV cache where models use it: the decode runner (steps in a CUDA graph, a prompt in one pass) against a 64-bit forward pass
over quantised pages, and the Hugging Face cache against a model whose attention quantises keys and values itself."""
import math

import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu


def _forward(m, tokens):
    """logits float64 [T, vocab] of one sequence, token by token: the runner's function over kv8_ref's pages, without its BF16 roundings"""
    c, D = m.cfg, m.cfg.head_dim
    W = lambda layer: layer.dequantize().cpu().double()                                       # noqa: E731
    blocks = []
    for qkv, o, gu, d in m.blocks:
        g = W(gu)
        if m.fused_act:
            g = g.view(c.inter // 16, 2, 16, c.hidden).transpose(0, 1).reshape(2 * c.inter, c.hidden)
        blocks.append((W(qkv), W(o), g, W(d)))
    embed, head, cos, sin = W(m.embed), W(m.lm_head), m.cos.cpu().double(), m.sin.cpu().double()
    one, ones = torch.ones(D), torch.ones(c.hidden)
    pages = [R.Pages(-(-len(tokens) // 16), m.hkv, D) for _ in blocks]
    out = []
    for t, tok in enumerate(tokens):
        x = embed[tok]
        for li, (qkv, o, gu, d) in enumerate(blocks):
            q, k, v = (qkv @ R.norm(x, ones, c.eps)).view(-1, D).split([m.hq, m.hkv, m.hkv])
            q, k = (R.rotate(R.norm(y, one, c.eps), cos[t], sin[t], True) for y in (q, k))
            pages[li].append(k[None], v[None], torch.tensor([t]))
            K, V = (y.flatten(0, 1) for y in pages[li].dense())
            x = x + o @ R.attend(q[None], K, V, [t], 1 / math.sqrt(D))[0].flatten()
            g, u = (gu @ R.norm(x, ones, c.eps)).chunk(2)
            x = x + d @ (torch.nn.functional.silu(g) * u)
        out.append(head @ R.norm(x, ones, c.eps))
    return torch.stack(out)


# Two layers of about ten roundings to BF16 (2^-8 each) on the way of a value: 20 * 2^-8 = 7.8e-2 at most; and a value that a rounding
# moves across a border of e4m3 moves by a step of 2^-3: one in 2^-8 / 2^-3 = 1/32 does, sqrt(1/32) * 2^-3 = 2.2e-2 in the mean square
REL = 0.1


@pytest.mark.parametrize("batch", [1, 3])
def test_decoder_steps_and_prefill(batch):
    from statetree_b200 import ops
    from statetree_b200.decoder import DecoderConfig, TreeDecoder
    cfg = DecoderConfig(layers=2, hidden=512, heads=4, kv_heads=2, head_dim=128, inter=1024, vocab=2048)
    P, new = 21, 6
    m = TreeDecoder(cfg, "cuda", batch, P + new + 8, seed=5, eight_bit_kv=True)
    prompt = torch.randint(0, cfg.vocab, (batch, P), generator=torch.Generator().manual_seed(2)).cuda()
    want = [_forward(m, prompt[b].tolist()) for b in range(batch)]
    m.capture()
    steps = []
    for t in range(P):
        m.tokens.copy_(prompt[:, t])
        m.graph.replay()
        steps.append(m.logits.cpu().double())
    by_step = [layer.dense() for layer in m.cache.layers]
    m.reset()
    whole = m.prefill(prompt[:, :16]).cpu().double(), m.prefill(prompt[:, 16:]).cpu().double()      # (in two chunks)
    m.cache.check()
    rel = lambda a, b: float((a - b).norm() / b.norm())                                       # noqa: E731
    for b in range(batch):
        assert rel(torch.stack([s[b] for s in steps]), want[b]) < REL
        assert rel(whole[0][b], want[b][15]) < REL and rel(whole[1][b], want[b][P - 1]) < REL
    for (k0, v0), layer in zip(by_step, m.cache.layers):
        k1, v1 = layer.dense()
        assert rel(k1.double(), k0.double()) < REL and rel(v1.double(), v0.double()) < REL
    # a prompt in one pass, then steps from the graph: the same tokens from run to run
    runs = []
    for _ in range(2):
        m.reset()
        runs.append(m.run(prompt, new))
        assert int(m.cache.cum) == P + new == int(m.pos_buf)
    assert torch.equal(runs[0], runs[1])
    m.reset()
    assert m.run(prompt, new, collect=[]).shape == (batch, new)
    with pytest.raises(ValueError, match="capacity"):
        m.prefill(prompt)
    with pytest.raises(ValueError, match="sequences"):
        m.prefill(prompt[:1].expand(batch + 1, P))
    with pytest.raises(ValueError, match="no tokens"):
        m.prefill(prompt[:, :0])
    assert ops.device_status() == 0


def test_decoder_with_experts_prefills():
    from statetree_b200.decoder import DecoderConfig, TreeDecoder
    cfg = DecoderConfig(layers=2, hidden=512, heads=4, kv_heads=1, head_dim=128, vocab=1024, experts=8, top_k=2, moe_inter=256)
    m = TreeDecoder(cfg, "cuda", 2, 64, seed=1, eight_bit_kv=True)
    m.capture()
    prompt = torch.randint(0, cfg.vocab, (2, 33), generator=torch.Generator().manual_seed(3)).cuda()
    for t in range(33):
        m.tokens.copy_(prompt[:, t])
        m.graph.replay()
    steps = m.logits.double()
    m.reset()
    whole = m.prefill(prompt).double()
    assert float((whole - steps).norm() / steps.norm()) < 2 * REL      # (both with the roundings above)


def test_prefill_is_refused_without_the_cache():
    from statetree_b200.decoder import DecoderConfig, TreeDecoder
    m = TreeDecoder(DecoderConfig(layers=1, hidden=256, heads=2, kv_heads=1, inter=256, vocab=256), "cuda", 1, 32)
    with pytest.raises(RuntimeError, match="eight_bit_kv"):
        m.prefill(torch.zeros(1, 4, dtype=torch.long, device="cuda"))


@pytest.mark.parametrize("head_dim", [64, 128])
@pytest.mark.parametrize("windows", [None, ["sliding_attention", "full_attention"], ["full_attention", "sliding_attention"]])
@pytest.mark.parametrize("pad", [0, 5])
def test_hf_cache(head_dim, windows, pad):
    """prompt in two chunks (longer than the windows of the layers that have one) and decode steps, one sequence left-padded, against
    a cache-free pass whose attention quantises by pages"""
    pytest.importorskip("transformers")
    from transformers import AttentionInterface, Qwen3Config, Qwen3ForCausalLM
    from transformers.integrations.sdpa_attention import sdpa_attention_forward
    from transformers.masking_utils import AttentionMaskInterface, sdpa_mask
    from statetree_b200.kvcache import StateTreeKVCache, enable
    cfg = Qwen3Config(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=head_dim, max_position_embeddings=256, tie_word_embeddings=False,
                      **(dict(use_sliding_window=True, sliding_window=8, layer_types=windows) if windows else {}))
    torch.manual_seed(0)
    model = Qwen3ForCausalLM(cfg).to(torch.bfloat16).cuda().eval()

    def quantised(t):
        B, H, T, D = t.shape
        pages = R.Pages(B * -(-T // 16), H, D)
        x = t.transpose(1, 2).reshape(B * T, H, D).cpu().double()
        pos = torch.arange(T)
        slots = (torch.arange(B)[:, None] * (-(-T // 16) * 16) + pos).flatten()
        pages.append(x, x, slots)
        return pages.dense()[0].flatten(0, 1)[slots].view(B, T, H, D).transpose(1, 2).to(t)

    def attention(module, query, key, value, mask, **kw):
        return sdpa_attention_forward(module, query, quantised(key), quantised(value), mask, **kw)

    AttentionInterface.register("kv8_plain", attention)
    AttentionMaskInterface.register("kv8_plain", sdpa_mask)
    B, P, steps = 2, 21, 6
    ids = torch.randint(0, cfg.vocab_size, (B, P + steps), device="cuda")
    mask = torch.ones(B, P + steps, dtype=torch.long, device="cuda")
    mask[1, :pad] = 0
    with torch.no_grad():
        model.set_attn_implementation("kv8_plain")
        full = model(input_ids=ids, attention_mask=mask).logits.float()
        enable(model)
        cache = StateTreeKVCache(model.config, batch_size=B, max_cache_len=P + steps + 8, eight_bit=True)
        got = []
        for a, b in [(0, 17), (17, P)] + [(P + t, P + t + 1) for t in range(steps - 1)]:
            out = model(input_ids=ids[:, a:b], attention_mask=mask[:, :b], past_key_values=cache, use_cache=True)
            got.append((b, out.logits[:, -1].float()))
    cache.check()
    assert cache.storage_bytes() == 2 * B * 3 * 2 * (2 * 16 * head_dim + 2)
    for n, g in got:
        want = full[:, n - 1]
        assert float((g - want).norm() / want.norm()) < REL, n
    k0, _ = cache.layers[0].dense(P)
    assert k0.shape == (B, 2, P, head_dim) and torch.isfinite(k0.float()).all()
    # the same cache again, for a prompt without padding: as a new one
    cache.reset()
    with torch.no_grad():
        one, two = (model(input_ids=ids[:, :7], past_key_values=c, use_cache=True).logits
                    for c in (cache, StateTreeKVCache(model.config, batch_size=B, max_cache_len=P + steps + 8, eight_bit=True)))
    assert torch.equal(one, two)
