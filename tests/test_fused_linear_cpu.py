"""What the products with an epilogue refuse before anything is launched (no GPU)."""
import ctypes

import pytest
import torch


def test_refusals_of_the_library():
    from statetree_b200 import ops
    L, p = ops.lib(), ctypes.c_void_p(4096)

    def gemm(B=4, M=128, N=64, act=0, res=None, stride=128, X=p, Y=p):
        return L.st_gemm_epilogue(p, p, p, X, Y, None, act, res, stride, B, M, N, None)

    def gemv(B=4, M=128, N=64, act=0, res=None, stride=128, X=p, Y=p):
        return L.st_gemv_epilogue(p, p, p, p, X, Y, None, act, res, stride, B, M, N, None, 0, None)
    odd = ctypes.c_void_p(4100)
    for call in (gemm, gemv):
        for bad, text in ((dict(M=120), b"M %"), (dict(N=65), b"N %"), (dict(B=0), b"batch"), (dict(act=6), b"activation"), (dict(act=-1), b"activation"),
                          (dict(act=5, M=48), b"SwiGLU"), (dict(res=p, stride=127), b"residual"), (dict(res=p, stride=130), b"residual"),
                          (dict(res=odd, stride=128), b"residual"), (dict(X=None), b"null"), (dict(Y=None), b"null"),
                          (dict(X=ctypes.c_void_p(4104)), b"16-byte")):
            assert call(**bad) != 0 and text in L.st_last_error(), (call, bad, L.st_last_error())
    assert gemv(B=33) != 0 and b"batch" in L.st_last_error()
    assert gemv(B=9, act=5) != 0 and b"8 rows" in L.st_last_error()


def test_refusals_of_the_layer():
    from statetree_b200 import TreeLinear
    tl = TreeLinear.from_weight(torch.randn(48, 64).to(torch.bfloat16))
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="activation"):
        tl.fused(x, "tanh")
    with pytest.raises(ValueError, match="pairs"):
        tl.fused(x, "swiglu")
    with pytest.raises(RuntimeError, match="CUDA"):
        tl.fused(x)


def test_spans():
    from statetree_b200.linear import _span
    t = torch.zeros(4, 6, dtype=torch.bfloat16)
    assert _span(t) == (t.data_ptr(), t.data_ptr() + 48) and _span(t[1:, :2]) == (t.data_ptr() + 12, t.data_ptr() + 40)
    first, last = _span(t[:0])
    assert first == last
