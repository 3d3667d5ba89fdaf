"""8-bit KV pages: what the attentions refuse about a block table with a row stride of its own, before any launch."""
import ctypes

import pytest

from test_kv8_cpu import P, _ops


def _attn(L, chunk, B=2, T=2, btw=4, bts=4, bt=P):
    if chunk:
        return L.st_kv8_chunk_attn_table(P, 512, T, 4, None, B, P, P, 4, 2, 128, bt, btw, bts, P, None, 0, P, 512, None, None, 0.1, 1, None)
    return L.st_kv8_attn_table(P, 512, B, 4, P, P, 4, 2, 128, bt, btw, bts, P, None, 0, P, 512, None, None, 0.1, 1, 1, None)


@pytest.mark.parametrize("chunk", [False, True])
@pytest.mark.parametrize("kw,word", [(dict(btw=0), b"block table"), (dict(btw=-1), b"block table"), (dict(bts=-4), b"block table"),
                                     (dict(btw=1 << 27), b"too large"), (dict(bt=None), b"null"), (dict(bt=ctypes.c_void_p(0)), b"null")])
def test_block_tables_refused(chunk, kw, word):
    L = _ops().lib()
    assert _attn(L, chunk, **kw) != 0
    assert word in L.st_last_error(), L.st_last_error()
    assert _attn(L, chunk, B=0, T=0) == 0
