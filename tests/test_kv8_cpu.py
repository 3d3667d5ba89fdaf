"""8-bit KV pages: what is refused, on the CPU: by the C entry points before any launch, and by the Python calls."""
import ctypes

import pytest
import torch


def _ops():
    from test_abi import _built
    return _built()


P = ctypes.c_void_p(4096)                                # (an address that no refused call follows)


def _append(L, N=1, H=2, D=128, ks=256, vs=256, K=P, blocks=4, pos=None, step=1, cos=None, sin=None, span=0, Q=None, qs=256, q_out=None,
            marks=None):
    return L.st_kv8_append(K, P, ks, vs, P, N, H, D, P, P, blocks, pos, step, cos, sin, span, 1, None, Q, qs, None, 2, q_out, 256, 1e-6,
                           marks, P, None)


def _attn(L, chunk=False, B=1, T=1, Hq=4, H=2, D=128, blocks=4, bts=4, q=P, window=0, scale=0.1, S=1, qs=512, wo=None):
    if chunk:
        return L.st_kv8_chunk_attn(q, qs, T, Hq, None, B, P, P, blocks, H, D, P, bts, P, None, window, P, 512, wo, wo, scale, S, None)
    return L.st_kv8_attn(q, qs, B, Hq, P, P, blocks, H, D, P, bts, P, None, window, P, 512, wo, wo, scale, S, 1, None)


def test_page_bytes():
    L = _ops().lib()
    assert L.st_kv8_page_bytes(8, 128) == 8 * 2 * 16 * 128 and L.st_kv8_page_bytes(1, 64) == 2048


@pytest.mark.parametrize("kw,word", [
    (dict(D=96), b"64 or 128"), (dict(N=-1), b"negative"), (dict(ks=260), b"multiples of 8"), (dict(K=ctypes.c_void_p(4104)), b"aligned"),
    (dict(K=None), b"null"), (dict(cos=P), b"both tables"), (dict(cos=P, sin=P, span=9), b"positions"), (dict(cos=P, sin=P, pos=P, span=0), b"positions"),
    (dict(cos=P, sin=P, pos=P, span=9, step=2), b"pos_step"), (dict(Q=P), b"queries"), (dict(Q=P, q_out=P, qs=4), b"queries"),
    (dict(N=385), b"marks")])
def test_append_refuses(kw, word):
    L = _ops().lib()
    assert _append(L, **kw) != 0
    assert word in L.st_last_error(), L.st_last_error()


@pytest.mark.parametrize("chunk", [False, True])
@pytest.mark.parametrize("kw,word", [
    (dict(D=80), b"64 or 128"), (dict(Hq=3), b"heads"), (dict(scale=0.0), b"scale"), (dict(scale=-1.0), b"scale"), (dict(scale=float("nan")), b"scale"),
    (dict(window=-1), b"window"), (dict(S=0), b"splits"), (dict(S=16), b"workspace"), (dict(q=None), b"null"), (dict(blocks=0), b"empty"),
    (dict(qs=4), b"multiples of 8"), (dict(q=ctypes.c_void_p(4100)), b"aligned")])
def test_attention_refuses(chunk, kw, word):
    L = _ops().lib()
    assert _attn(L, chunk, **kw) != 0
    assert word in L.st_last_error(), L.st_last_error()


def test_outputs_whose_rows_overlap_are_refused():
    L = _ops().lib()
    assert _attn(L, B=2, T=2, Hq=8, qs=0) != 0 and b"overlap" in L.st_last_error()
    assert _attn(L, True, B=1, T=5, Hq=8, qs=0) != 0 and b"overlap" in L.st_last_error()
    assert L.st_kv8_append(P, P, 256, 256, P, 2, 2, 128, P, P, 4, None, 1, None, None, 0, 1, None, P, 0, None, 4, P, 256, 1e-6, None, P, None) != 0
    assert b"overlap" in L.st_last_error()


def test_workspace_of_split_attentions():
    """none where the splits join on chip (two to eight of them, about a wave of CTAs), else a partial row per split"""
    ws = _ops().lib().st_kv8_attn_workspace_bytes
    assert ws(1, 1, 32, 8, 128, 1, 0) == ws(1, 1, 32, 8, 128, 8, 0) == ws(0, 0, 32, 8, 128, 4, 1) == 0
    assert ws(1, 1, 32, 8, 128, 9, 0) == 32 * 9 * 130 * 4
    assert ws(64, 64, 32, 8, 64, 2, 0) == 64 * 32 * 2 * 66 * 4 and ws(32, 32, 32, 8, 64, 2, 0) == 0
    assert ws(32, 8, 32, 8, 128, 4, 1) == 0                                     # eight sequences of four queries: 512 CTAs of eight rows
    assert ws(100, 1, 32, 8, 128, 2, 1) == 100 * 32 * 2 * 130 * 4               # (the tensor-core kernel)


def test_empty_calls_are_no_calls():
    L = _ops().lib()
    assert _append(L, N=0) == 0 and _attn(L, B=0) == 0 and _attn(L, True, T=0, B=0) == 0
    assert L.st_kv8_dequant_blocks(P, P, 4, 2, 128, P, 0, P, P, None) == 0
    assert L.st_kv8_chunk_attn(P, 512, 2, 4, None, 1, P, P, 4, 2, 128, P, 4, P, None, 0, P, 512, None, None, 0.1, 1, None) != 0
    assert b"one query" in L.st_last_error()
    assert L.st_kv8_dequant_blocks(P, P, 4, 2, 128, None, 5, P, P, None) != 0 and b"more pages" in L.st_last_error()


def test_python_calls_refuse():
    _ops()
    from statetree_b200.kvcache import PageStore8
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)                                     # noqa: E731
    with pytest.raises(RuntimeError, match="64 or 128"):
        PageStore8(4, 2, "cpu", head_dim=96)
    with pytest.raises(RuntimeError, match="exponents"):
        PageStore8.over(torch.zeros(4, 2, 2, 16, 64, dtype=torch.uint8), torch.zeros(4, 2, dtype=torch.int8))
    s = PageStore8(4, 2, "cpu")
    slots = torch.zeros(3, dtype=torch.int64)
    K = bf(3, 2, 128)
    with pytest.raises(RuntimeError, match="CUDA tensors only"):
        s.append(K, K, slots)
    for bad, word in ((dict(K=bf(3, 2, 64)), "K BF16"), (dict(K=bf(3, 1, 128), V=bf(3, 1, 128)), "heads"), (dict(V=bf(2, 2, 128)), "heads"),
                      (dict(K=torch.zeros(3, 2, 128)), "K BF16"), (dict(slots=slots[:2]), "slots"), (dict(slots=slots.int()), "slots"),
                      (dict(cos=torch.zeros(9, 64)), "rotation"), (dict(cos=torch.zeros(9, 64), sin=torch.zeros(9, 64)), "rotation"),
                      (dict(cos=torch.zeros(9, 32), sin=torch.zeros(9, 32), positions=slots), "cos and sin"),
                      (dict(cos=torch.zeros(9, 64), sin=torch.zeros(9, 64), positions=slots[:2]), "positions"),
                      (dict(k_norm=bf(64)), "norm weights"), (dict(q=bf(2, 4, 128)), "Q and q_out")):
        with pytest.raises(RuntimeError, match=word):
            s.append(**{**dict(K=K, V=K, slots=slots), **bad})
    table, lens = torch.zeros(3, 4, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)
    q = bf(3, 4, 128)
    for bad, word in ((dict(q=bf(3, 3, 128)), "multiple of 2"), (dict(q=bf(2, 4, 128)), "one query"), (dict(lens=lens.long()), "lens"),
                      (dict(lens=lens[:2]), "lens"), (dict(block_table=table.long()), "block table"), (dict(starts=lens[:1]), "starts"),
                      (dict(window=-1), "window"), (dict(splits=0), "splits"), (dict(out=bf(3, 2, 128)), "out"), (dict(q=q.float()), "q BF16")):
        with pytest.raises(RuntimeError, match=word):
            s.attention(**{**dict(q=q, block_table=table, lens=lens, scale=0.1), **bad})
    with pytest.raises(RuntimeError, match="cu int32"):
        s.chunk_attention(q, lens, table, lens, 0.1)
    with pytest.raises(RuntimeError, match="one query"):
        s.chunk_attention(bf(5, 4, 128), None, table, lens, 0.1)
    with pytest.raises(RuntimeError, match="blocks"):
        from statetree_b200.ops import kv_ext
        kv_ext().kv8_dequant_blocks(s.pages, s.exps, torch.zeros(2, dtype=torch.int64), bf(2, 16, 2, 128), bf(2, 16, 2, 128))


def test_paged_cache_chunks():
    """slots and lengths of whole chunks, and what does not fit"""
    _ops()
    from statetree_b200.kvcache import PagedKVCache, PageStore8
    c = PagedKVCache(2, 2, 40, 3, "cpu", eight_bit=True, head_dim=64)
    assert all(isinstance(layer, PageStore8) and layer.pages.shape == (6, 3, 2, 16, 64) for layer in c.layers)
    assert c.begin_chunk(2, 20).tolist() == list(range(20)) + list(range(48, 68)) and c.lens.tolist() == [20, 20]
    c.end_chunk(20)
    assert c.begin_chunk(2, 5).tolist() == list(range(20, 25)) + list(range(68, 73)) and c.lens.tolist() == [25, 25]
    with pytest.raises(ValueError, match="capacity"):
        c.begin_chunk(2, 29)
    c.layers[0].bad.fill_(1)
    with pytest.raises(RuntimeError, match="finite"):
        c.check()
    c.reset()
    c.check()
    assert int(c.cum) == 0 and c.begin_chunk(2, 48).numel() == 96


def test_split_rules():
    """as many splits as the rules state, never more than pages allow"""
    _ops()
    from statetree_b200.kvcache import chunk_splits8, decode_splits8
    assert decode_splits8(8, 1000) == 18 and decode_splits8(8, 63) == 8 and decode_splits8(8, 19) == 2 and decode_splits8(1, 4) == 1
    assert decode_splits8(64, 1000) == 8 and decode_splits8(512, 512) == 4 and decode_splits8(512, 100) == 1 and decode_splits8(4096, 512) == 2
    assert chunk_splits8(4096, 1, 8, 4, 256) == 1 and chunk_splits8(16, 1, 8, 4, 250) == 15 and chunk_splits8(4, 1, 8, 4, 250) == 8
    for units in range(1, 700, 7):
        for pages in (1, 2, 7, 33, 500, 5000):
            assert 1 <= decode_splits8(units, pages) <= max(1, min(64, pages // 6))
