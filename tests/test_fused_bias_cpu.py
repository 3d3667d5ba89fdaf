"""What the products with an epilogue take for a bias (no GPU): BF16, a value a row; anything else is refused before a pointer is looked at."""
import pytest
import torch


@pytest.mark.parametrize("bias", [torch.zeros(48), torch.zeros(48, dtype=torch.float16), torch.zeros(32, dtype=torch.bfloat16),
                                  torch.zeros(48, 1, dtype=torch.bfloat16), torch.zeros(96, dtype=torch.bfloat16)[::2],
                                  torch.zeros(48, dtype=torch.bfloat16, device="meta"), torch.zeros(48, dtype=torch.uint8)],
                         ids=["fp32", "fp16", "short", "2d", "strided", "elsewhere", "bytes"])
def test_a_bias_that_is_not_read_as_it_is(bias):
    from statetree_b200.ops import ext
    tree, x, y = torch.zeros(3, 1, 1552, dtype=torch.uint8), torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(2, 48, dtype=torch.bfloat16)
    i = torch.zeros(16, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="bias BF16"):
        ext().gemv_epilogue(tree, i, i, i, x, y, bias, 0, None, torch.zeros(16))
    with pytest.raises(RuntimeError, match="bias BF16"):
        ext().gemm_epilogue(tree, i, i, x, y, bias, 0, None)


def test_the_bias_that_is():
    """... is looked at no further: the refusal is the one of tensors that are not on a GPU"""
    from statetree_b200.ops import ext
    tree, x, y = torch.zeros(3, 1, 1552, dtype=torch.uint8), torch.zeros(2, 64, dtype=torch.bfloat16), torch.zeros(2, 48, dtype=torch.bfloat16)
    i = torch.zeros(16, dtype=torch.int32)
    for bias in (None, torch.zeros(48, dtype=torch.bfloat16)):
        with pytest.raises(RuntimeError, match="CUDA"):
            ext().gemm_epilogue(tree, i, i, x, y, bias, 0, None)
