"""What the chunk attention over lossless pages refuses before it launches anything, and how it is split (no GPU)."""
import ctypes

import pytest


def test_refusals_of_the_library():
    from statetree_b200 import ops
    L, p = ops.lib(), ctypes.c_void_p(4096)

    def call(T=4, Hq=4, B=2, cu=p, Hkv=2, qs=512, q=p, pool=p, btw=3, window=0, os=512, wo=None, scale=1.0, S=1, nblocks=9, whole=0):
        return L.st_kv_chunk_attn(q, qs, T, Hq, cu, B, p, nblocks, Hkv, pool, 8, p, btw, btw, p, None, window, p, os, wo, wo, scale, S, whole, None)
    for bad, text in ((dict(Hq=3), b"heads"), (dict(scale=0.0), b"scale"), (dict(window=-1), b"window"), (dict(q=None), b"null"),
                      (dict(pool=None), b"null"), (dict(qs=511), b"multiples of 8"), (dict(os=504), b"overlap"), (dict(S=0), b"splits"), (dict(whole=-1), b"splits"),
                      (dict(S=2), b"workspace"), (dict(S=2000, wo=p), b"splits"), (dict(cu=None), b"one query"), (dict(btw=0), b"empty"),
                      (dict(nblocks=1 << 31), b"pages"), (dict(q=ctypes.c_void_p(4104)), b"aligned")):
        assert call(**bad) != 0 and text in L.st_last_error(), (bad, L.st_last_error())
    assert call(T=0) == 0 and call(B=0) == 0
    assert L.st_kv_chunk_attn_workspace_bytes(10, 4, 1) == 0 and L.st_kv_chunk_attn_workspace_bytes(10, 4, 3) == 10 * 4 * 3 * 130 * 4


@pytest.mark.parametrize("tokens,seqs,kv,group,pages", [(1, 1, 8, 4, 1), (4096, 1, 8, 4, 256), (2048, 1, 8, 4, 2003), (32, 8, 8, 4, 182),
                                                        (0, 3, 1, 1, 9), (5, 0, 2, 2, 9), (64, 64, 1, 64, 4000)])
def test_splits(tokens, seqs, kv, group, pages):
    from statetree_b200.kvcache import chunk_splits
    n, whole = chunk_splits(tokens, seqs, kv, group, pages)
    assert 1 <= n <= 64 and n <= max(1, pages) and whole >= 0 and (n > 1 or whole == 0)


def test_splits_of_a_last_wave():
    """256 units of equal length on 148 SMs: the first 148 whole, behind the eight that have no rows; a prompt from its beginning as it is"""
    from statetree_b200.kvcache import chunk_splits
    n, whole = chunk_splits(2048, 1, 8, 4, 2003)
    assert n > 1 and whole == 148 + 8
    assert chunk_splits(4096, 1, 8, 4, 256) == (1, 0)


def test_pages_are_checked():
    import torch
    from statetree_b200.kvcache import PageStore
    ok = torch.zeros(2, 1, 2, 2, 1600, dtype=torch.uint8)
    pool = torch.zeros(4, 16, dtype=torch.int32)
    assert PageStore.over(ok, pool).pcnt.tolist() == [4, 0]
    for pages, pl in ((ok.int(), pool), (ok[0], pool), (ok[..., :1598], pool), (ok, pool.long()), (ok, pool[:, :15])):
        with pytest.raises(RuntimeError):
            PageStore.over(pages, pl)
    with pytest.raises(RuntimeError):
        PageStore.over(ok, pool, torch.zeros(3, dtype=torch.int32))
