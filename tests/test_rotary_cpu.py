"""Tables of the rotary positions, and what the rotation refuses before it launches anything (no GPU)."""
import ctypes
import math

import pytest
import torch

from statetree_b200.rotary import rotary_tables


def test_plain_table_far_out():
    """positions beyond 2^24: the angles are formed in 64 bits, so a table's row is the cosine of that very position"""
    part, theta = 64, 1e4
    cos, sin = rotary_tables(part, 1 << 12, theta, device="cpu")
    p = torch.tensor([0, 1, 4095], dtype=torch.float64)
    ang = p[:, None] * theta ** (-torch.arange(0, part, 2, dtype=torch.float64) / part)
    assert cos.shape == sin.shape == (1 << 12, part // 2) and cos.dtype == torch.float32
    assert float((cos[p.long()] - ang.cos()).abs().max()) < 2.0 ** -24 and float((sin[p.long()] - ang.sin()).abs().max()) < 2.0 ** -24
    one = rotary_tables(2, (1 << 23) + 3, 1e4, device="cpu")[0][-1, 0]     # (made in several parts)
    assert abs(float(one) - math.cos((1 << 23) + 2)) < 2.0 ** -24


@pytest.mark.parametrize("scaling", [
    dict(rope_type="default"), dict(rope_type="linear", factor=4.0), dict(type="linear", factor=2.5),
    dict(rope_type="dynamic", factor=2.0, original_max_position_embeddings=512),
    dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=512),
    dict(rope_type="yarn", factor=4.0, original_max_position_embeddings=512, beta_fast=16.0, beta_slow=2.0, attention_factor=1.25),
    dict(rope_type="llama3", factor=8.0, original_max_position_embeddings=512, low_freq_factor=1.0, high_freq_factor=4.0),
    dict(rope_type="longrope", factor=4.0, original_max_position_embeddings=512, short_factor=[1.0 + 0.1 * i for i in range(32)],
         long_factor=[1.0 + i for i in range(32)]),
], ids=lambda s: s.get("rope_type", s.get("type")))
def test_scaled_tables_agree_with_the_models(scaling):
    """the frequencies that Hugging Face models make of the same configuration (theirs are float32: 2^-20 of an angle up to 600)"""
    pytest.importorskip("transformers")
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    length, theta, part = 600, 1e4, 64
    cos, sin = rotary_tables(part, length, theta, scaling, device="cpu")
    kind = scaling.get("rope_type", scaling.get("type"))
    if kind == "default":
        inv, amp = theta ** (-torch.arange(0, part, 2).double() / part), 1.0
    else:
        sc = dict(scaling, rope_type=kind, rope_theta=theta)
        cfg = LlamaConfig(hidden_size=256, num_attention_heads=4, head_dim=part, max_position_embeddings=length if kind == "longrope" else 512,
                          rope_parameters=sc)
        if kind == "longrope":
            cfg.original_max_position_embeddings = 512
        inv, amp = ROPE_INIT_FUNCTIONS[kind](cfg, "cpu", seq_len=length)
    ang = torch.arange(length).double()[:, None] * inv.double()
    assert float((cos - ang.cos() * amp).abs().max()) < 600 * 2.0 ** -20 and float((sin - ang.sin() * amp).abs().max()) < 600 * 2.0 ** -20


@pytest.mark.parametrize("args", [(63, 8), (0, 8), (64, 0), (64, 8, 1e4, dict(rope_type="yarn", factor=2.0)),
                                  (64, 8, 1e4, dict(rope_type="linear")), (64, 8, 1e4, dict(rope_type="linear", factor=0.5)),
                                  (64, 8, 1e4, dict(rope_type="none such")),
                                  (64, 8, 1e4, dict(rope_type="longrope", original_max_position_embeddings=4, long_factor=[1.0]))])
def test_tables_refuse(args):
    with pytest.raises(ValueError):
        rotary_tables(*args, device="cpu")


def test_refusals_of_the_library():
    from statetree_b200 import ops
    L, p = ops.lib(), ctypes.c_void_p(4096)

    def call(N=1, D=64, kind=0, part=64, offset=0, span=8, q=p, pos=p):
        return L.st_rotate(q, 64, 64, 1, None, 0, 0, 0, N, D, kind, pos, 1, p, p, span, part, offset, 1, 0, None, None, 1e-6, p, 64, 64, None, 0,
                           0, None)
    for bad, text in ((dict(kind=3), b"type"), (dict(part=63), b"even"), (dict(part=62, offset=4), b"even"), (dict(span=0), b"table"),
                      (dict(q=None), b"null"), (dict(pos=None), b"null"), (dict(N=-1), b"sizes")):
        assert call(**bad) != 0 and text in L.st_last_error(), (bad, L.st_last_error())
    assert call(N=0) == 0                                    # (nothing to do, nothing launched)


def test_refusals_of_the_call():
    from statetree_b200.rotary import rotate
    q = torch.zeros(2, 1, 64, dtype=torch.bfloat16)
    c = torch.zeros(4, 32)
    with pytest.raises(RuntimeError, match="CUDA"):
        rotate(q, None, torch.zeros(2, dtype=torch.long), c, c)
    w = torch.ones(64, dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="gradients"):
        rotate(q.requires_grad_(), None, torch.zeros(2, dtype=torch.long), c, c, q_norm=w)


def test_outputs_apart():
    """which rows share values: parts of one fused buffer lie apart, overlapping ones do not"""
    from statetree_b200.ops import _Weights
    buf = torch.zeros(10, 8, 16)
    apart = _Weights._apart
    assert apart(buf[:, :3], buf[:, 3:5]) and apart(buf[:, 3:5], buf[:, :3]) and apart(buf[:5], buf[5:])
    assert not apart(buf[:, :3], buf[:, 2:5]) and not apart(buf, buf) and not apart(buf[:, :3], buf[1:, :3])
    assert not apart(buf[:, :, :8], buf[:, :, 4:12])
    assert apart(buf[:0], buf) and apart(torch.zeros(10, 8, 16), buf)


def test_output_layouts():
    """rows whose values have memory of their own, whichever of token and head lies further apart; shared ones are told"""
    from statetree_b200.ops import _Weights
    own = _Weights._own_memory
    buf = torch.zeros(6, 10, 16)
    assert own(buf) and own(buf.transpose(0, 1)) and own(buf[:, ::2]) and own(buf[:, :, :8]) and own(buf.transpose(0, 1)[:, 1:4])
    assert own(buf[:1].expand(1, 10, 16)) and own(buf[:0]) and own(buf[:, :1].as_strided((6, 1, 16), (160, 0, 1)))
    assert not own(buf[:, :1].expand(6, 10, 16)) and not own(buf[:1].expand(6, 10, 16)) and not own(buf.as_strided((6, 4, 16), (32, 16, 1)))
    assert not own(buf.as_strided((6, 4, 16), (16, 32, 1))) and not own(buf.as_strided((6, 4, 16), (64, 8, 1)))
