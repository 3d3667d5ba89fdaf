"""Tables of the rotary positions for the keys that model configurations carry beside the common ones: the tables that Hugging Face models make of
the same configuration, and refusals of what would make another table."""
import pytest
import torch

from statetree_b200.rotary import rotary_tables

PART, THETA = 64, 1e4


def models(scaling, length, max_length):
    """(cos, sin) in 64 bits of the frequencies and the amplitude of a model whose configuration has `scaling` and `max_length` positions"""
    pytest.importorskip("transformers")
    from transformers import LlamaConfig
    from transformers.modeling_rope_utils import ROPE_INIT_FUNCTIONS
    cfg = LlamaConfig(hidden_size=256, num_attention_heads=4, head_dim=PART, max_position_embeddings=max_length,
                      rope_parameters=dict({"rope_theta": THETA}, **scaling))
    inv, amp = ROPE_INIT_FUNCTIONS[scaling["rope_type"]](cfg, "cpu", seq_len=length)
    ang = torch.arange(length).double()[:, None] * inv.double()
    return ang.cos() * amp, ang.sin() * amp


def agree(got, want, amp=2.0):
    """theirs are float32 frequencies: each is off by some 2^-22 of itself (a power, a division, sums), the angle by as much of up to
    `length`, cosine and sine by as much as the angle, times the amplitude"""
    tol = amp * got[0].shape[0] * 2.0 ** -20
    assert all(float((g - w).abs().max()) < tol for g, w in zip(got, want))


@pytest.mark.parametrize("factor", [2.0, 32.0])
@pytest.mark.parametrize("truncate", [True, False])
def test_yarn_with_and_without_whole_pairs(truncate, factor):
    sc = dict(rope_type="yarn", factor=factor, original_max_position_embeddings=512, beta_fast=32.0, beta_slow=1.0, truncate=truncate)
    agree(rotary_tables(PART, 600, THETA, sc, device="cpu"), models(sc, 600, 512))


@pytest.mark.parametrize("more", [dict(mscale=1.0, mscale_all_dim=1.0), dict(mscale=0.707, mscale_all_dim=1.0), dict(mscale=0.707),
                                  dict(mscale_all_dim=0.707), dict(mscale=1.0, mscale_all_dim=0.0),
                                  dict(mscale=0.5, mscale_all_dim=1.0, attention_factor=1.3), dict(mscale=0.5, mscale_all_dim=1.0, factor=1.0)], ids=str)
def test_yarn_amplitudes(more):
    sc = {**dict(rope_type="yarn", factor=40.0, original_max_position_embeddings=512), **more}
    agree(rotary_tables(PART, 600, THETA, sc, device="cpu"), models(sc, 600, 512))


LONG = dict(rope_type="longrope", original_max_position_embeddings=512, short_factor=[1.0 + 0.1 * i for i in range(32)],
            long_factor=[1.0 + i for i in range(32)])


@pytest.mark.parametrize("length", [1, 300, 512, 513, 2000])
@pytest.mark.parametrize("max_length", [600, 8192])
def test_longrope_amplitude_is_the_models(max_length, length):
    """... and no table's: tables of any length of one model have the same amplitude, in the row of position 0"""
    got = rotary_tables(PART, length, THETA, dict(LONG, max_position_embeddings=max_length), device="cpu")
    agree(got, models(LONG, length, max_length))
    assert bool((got[0][0] == rotary_tables(PART, 4096, THETA, dict(LONG, max_position_embeddings=max_length), device="cpu")[0][0]).all())


@pytest.mark.parametrize("more", [dict(factor=4.0), dict(factor=4.0, attention_factor=1.7), dict(attention_factor=1.25), dict(factor=1.0)], ids=str)
def test_longrope_amplitudes(more):
    """a factor goes before the lengths, an attention factor before both"""
    sc = dict(LONG, **more)
    agree(rotary_tables(PART, 600, THETA, dict(sc, max_position_embeddings=8192), device="cpu"), models(sc, 600, 8192))
    agree(rotary_tables(PART, 600, THETA, sc, device="cpu"), models(sc, 600, 8192))


def test_longrope_needs_the_models_stretch():
    for length in (300, 2000):
        with pytest.raises(ValueError, match="max_position_embeddings"):
            rotary_tables(PART, length, THETA, LONG, device="cpu")


@pytest.mark.parametrize("sc", [dict(rope_type="llama3", factor=8.0, original_max_position_embeddings=512, low_freq_factor=1.0, high_freq_factor=4.0),
                                dict(rope_type="linear", factor=2.0), dict(LONG, factor=4.0),
                                dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=512)], ids=lambda s: s["rope_type"])
def test_theta_of_the_configuration(sc):
    """a configuration that keeps its base beside the scaling"""
    own = dict(sc, rope_theta=5e5)
    got = rotary_tables(PART, 600, scaling=own, device="cpu")
    agree(got, models(own, 600, 512))
    assert all(bool((a == b).all()) for a, b in zip(got, rotary_tables(PART, 600, 5e5, sc, device="cpu")))
    assert all(bool((a == b).all()) for a, b in zip(got, rotary_tables(PART, 600, 500000, own, device="cpu")))       # (the same, twice)


def test_theta_by_default_and_by_the_plain_kind():
    plain, base = rotary_tables(PART, 64, device="cpu"), rotary_tables(PART, 64, 1e4, device="cpu")
    assert all(bool((a == b).all()) for a, b in zip(plain, base))
    plain, base = rotary_tables(PART, 64, scaling=dict(rope_type="default", rope_theta=1e6), device="cpu"), rotary_tables(PART, 64, 1e6, device="cpu")
    assert all(bool((a == b).all()) for a, b in zip(plain, base))


def test_two_thetas_are_refused():
    with pytest.raises(ValueError, match="rope_theta"):
        rotary_tables(PART, 8, 1e4, dict(rope_type="default", rope_theta=5e5), device="cpu")


@pytest.mark.parametrize("sc", [
    dict(factor=2.0), dict(rope_type="default", mrope_section=[16, 24, 24]), dict(rope_type="linear", factor=2.0, mscale=1.0),
    dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=512, attn_factor=1.5),
    dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=512, finetuned=True), dict(LONG, factor=4.0, short_mscale=1.2),
    dict(full_attention=dict(rope_type="default"), sliding_attention=dict(rope_type="linear", factor=2.0))], ids=str)
def test_keys_that_are_not_read_are_refused(sc):
    """... they make another table in a model that reads them; a whole configuration of several kinds of layers is none of one kind"""
    with pytest.raises(ValueError, match="does not read|unknown rope_type"):
        rotary_tables(PART, 8, scaling=sc, device="cpu")


def test_keys_without_a_value_and_of_the_models_sizes():
    plain = rotary_tables(PART, 8, device="cpu")
    same = rotary_tables(PART, 8, scaling=dict(rope_type="default", mrope_section=None, factor=None, partial_rotary_factor=0.5,
                                               max_position_embeddings=4096), device="cpu")
    assert all(bool((a == b).all()) for a, b in zip(plain, same))
    sc = dict(rope_type="yarn", factor=8.0, original_max_position_embeddings=512)
    assert all(bool((a == b).all()) for a, b in zip(rotary_tables(PART, 8, scaling=sc, device="cpu"), rotary_tables(
        PART, 8, scaling=dict(sc, attention_factor=None, mscale=None, beta_fast=None, max_position_embeddings=4096), device="cpu")))


@pytest.mark.parametrize("length", [600, 1024, 1500])
def test_dynamic_counts_from_the_models_maximum(length):
    sc = dict(rope_type="dynamic", factor=2.0, original_max_position_embeddings=512)
    agree(rotary_tables(PART, length, THETA, dict(sc, max_position_embeddings=1024), device="cpu"), models(sc, length, 1024))
    agree(rotary_tables(PART, length, THETA, dict(rope_type="dynamic", factor=2.0, max_position_embeddings=1024), device="cpu"),
          models(sc, length, 1024))
