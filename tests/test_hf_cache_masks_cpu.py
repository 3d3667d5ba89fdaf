"""The Hugging Face cache on the CPU with a store that only takes notes: which masks its attention reads as left padding, and
which masks and modules it refuses over 8-bit pages."""
import types

import pytest
import torch

pytest.importorskip("transformers")
NEG = torch.finfo(torch.bfloat16).min


class _Notes:
    """a PageStore8's calls"""
    def __init__(self):
        self.calls = []

    def _take(self, kind, q, starts, window):
        self.calls.append((kind, starts.tolist(), window))
        return torch.zeros_like(q)

    def chunk_attention(self, q, cu, table, lens, scale, splits=None, starts=None, out=None, window=0):
        return self._take("chunk", q, starts, window)

    def attention(self, q, table, lens, scale, splits=None, starts=None, min_pages=4, out=None, window=0):
        return self._take("step", q, starts, window)

    def append(self, K, V, slots):
        pass

    def dense(self):
        return torch.zeros(2, 2 * 16, 16, 2, 128, dtype=torch.bfloat16)

    def reset(self):
        pass


class _Model:
    """layers of an attention module over one cache, fed mask by mask"""
    def __init__(self, B, layers=2, eight_bit=True):
        from statetree_b200.kvcache import StateTreeKVCache
        cfg = types.SimpleNamespace(num_hidden_layers=layers, num_attention_heads=4, num_key_value_heads=2)
        self.cache = StateTreeKVCache(cfg, batch_size=B, max_cache_len=256, eight_bit=eight_bit)
        self.B, self.notes = B, _Notes()

    def __call__(self, T, mask, windows=None, module=None, **kw):
        """a forward pass over T tokens; a mask and a window for all layers, or a list of them"""
        from statetree_b200.kvcache import statetree_attention
        of = lambda x, i: x[i] if isinstance(x, list) else x                                  # noqa: E731
        q, k = (torch.zeros(self.B, h, T, 128, dtype=torch.bfloat16) for h in (4 if self.cache.eight_bit else 2, 2))
        for i, layer in enumerate(self.cache.layers):
            if not layer.is_initialized:
                layer.lazy_initialization(k, k)
                layer.store = self.notes
            keys, values = layer.update(k, k)
            attends = types.SimpleNamespace(layer_idx=i, **{"is_causal": True, **(module or {})})
            statetree_attention(attends, q, keys, values, of(mask, i), scaling=0.1, sliding_window=of(windows, i), **kw)

    @property
    def starts(self):
        return self.notes.calls[-1][1]


def _mask(pads, before, T, window=0, kind="bool"):
    """[B, 1, T, before + T]: causal with left padding (and a window)"""
    K = before + T
    k, p = torch.arange(K), torch.arange(before, K)[:, None]
    m = (k <= p) & (k >= torch.tensor(pads)[:, None, None])
    if window:
        m &= k > p - window
    m = m[:, None]
    return m if kind == "bool" else torch.zeros(m.shape, dtype=torch.bfloat16).masked_fill(~m, -float("inf") if kind == "inf" else NEG)


@pytest.mark.parametrize("kind", ["bool", "inf", "lowest"])
@pytest.mark.parametrize("window", [0, 5, 40])
@pytest.mark.parametrize("pads", [[0, 3], [0, 20], [16, 33], [40, 1]])
def test_left_padding_longer_than_a_chunk(pads, window, kind):
    """chunks of 16: a sequence's padding may end in any of them"""
    m, at = _Model(2), 0
    for T in (16, 16, 16, 1, 7, 1):
        m(T, _mask(pads, at, T, window, kind), window or None)
        at += T
        seen = [min(p, at) for p in pads]
        assert m.starts == seen and m.notes.calls[-1][2] == window
    assert [c[0] for c in m.notes.calls] == ["chunk"] * 6 + ["step"] * 2 + ["chunk"] * 2 + ["step"] * 2
    m.cache.reset()
    m(3, None)
    assert m.starts == [0, 0]


@pytest.mark.parametrize("windows", [[None, 6], [6, None]])
def test_layers_with_and_without_a_window(windows):
    m = _Model(2)
    for at, T in ((0, 16), (16, 16), (32, 4)):
        m(T, [_mask([0, 21], at, T, w or 0) for w in windows], windows)
        assert m.starts == [0, min(21, at + T)]


@pytest.mark.parametrize("kind", ["bool", "inf"])
@pytest.mark.parametrize("pads", [[0, 3], [0, 20], [16, 33], [40, 1]])
def test_left_padding_of_the_lossless_cache(pads, kind):
    """decode steps begin behind the padding there too"""
    m, at = _Model(2, eight_bit=False), 0
    for T in (16, 16, 16, 1, 7, 1):
        m(T, _mask(pads, at, T, 0, kind))
        at += T
        assert m.cache.starts.tolist() == [min(p, at) for p in pads]
    assert m.notes.calls == [("step", pads, 0)] * 4


@pytest.mark.parametrize("kind", ["bool", "lowest"])
def test_rows_of_padding_may_see_everything(kind):
    """masks that leave no row empty let a padding token see everything"""
    mask = _mask([0, 3], 0, 8, kind=kind)
    mask[1, :, :3] = mask[0, 0, 7, 0]
    m = _Model(2)
    m(8, mask)
    assert m.starts == [0, 3]


def _packed():
    m = _mask([0, 0], 0, 8)
    m[:, :, 3:, :3] = False
    return m


def _right():
    return _mask([0, 0], 0, 8) & torch.tensor([[1] * 8, [1] * 6 + [0, 0]], dtype=torch.bool)[:, None, None]


def _prefix():
    m = _mask([0, 0], 0, 8)
    m[:, :, :4, :4] = True
    return m


def _holes():
    m = _mask([0, 0], 0, 8)
    m[1, 0, 7, 4] = False
    return m


def _heads():
    m = _mask([0, 0], 0, 8).repeat(1, 4, 1, 1)
    m[1, 2, 7, 4] = False
    return m


@pytest.mark.parametrize("make", [_packed, _right, _prefix, _holes, _heads])
@pytest.mark.parametrize("kind", [torch.bool, torch.float32])
def test_other_masks_are_refused(make, kind):
    """packed sequences, right padding, a prefix that sees ahead, single hidden keys, heads of their own"""
    mask = make()
    if kind != torch.bool:
        mask = torch.zeros(mask.shape).masked_fill(~mask, -float("inf"))
    with pytest.raises(ValueError, match="mask"):
        _Model(2)(8, mask)


@pytest.mark.parametrize("row", [0, 1, 70, 129, 130, 199])
def test_a_mask_is_checked_in_all_its_rows(row, monkeypatch):
    """large masks are gone through some rows at a time"""
    from statetree_b200 import hf_cache
    monkeypatch.setattr(hf_cache, "MASK_PART", 65 * 200 * 2)
    mask = _mask([0, 0], 0, 200)
    _Model(2)(200, mask)
    mask[1, 0, row, row] = False
    with pytest.raises(ValueError, match="mask"):
        _Model(2)(200, mask)


def test_more_masks_are_refused():
    bias = torch.zeros(2, 1, 8, 8).masked_fill(~_mask([0, 0], 0, 8), -float("inf"))
    bias[0, 0, 5, 2] = -0.5                                # a bias, not a mask
    nan = bias.clone()
    nan[0, 0, 5, 2] = float("nan")
    for mask in (bias, nan, _mask([0, 0], 0, 8, 4), _mask([0, 0], 0, 8)[:, 0], torch.ones(2, 8)):
        with pytest.raises(ValueError, match="mask"):
            _Model(2)(8, mask)
    with pytest.raises(ValueError, match="mask"):          # a window that the mask has not
        _Model(2)(8, _mask([0, 0], 0, 8), 4)
    m = _Model(2)                                          # only the second layer's, and only in a later pass
    m(8, _mask([0, 2], 0, 8))
    m(8, _mask([0, 2], 8, 8))
    late = _mask([0, 2], 16, 8)
    late[0, 0, 7, 9] = False
    with pytest.raises(ValueError, match="mask"):
        m(8, [_mask([0, 2], 16, 8), late])


@pytest.mark.parametrize("T", [4, 1])
@pytest.mark.parametrize("kw", [dict(softcap=30.0), dict(s_aux=torch.zeros(4)), dict(dropout=0.1)])
def test_attention_of_another_kind_is_refused(T, kw):
    m = _Model(1)
    m(3, None)
    with pytest.raises(ValueError, match=next(iter(kw))):
        m(T, None, **kw)
    for off in (dict(softcap=None, s_aux=None, dropout=0.0), dict(softcap=0.0, dropout=None)):
        _Model(1)(4, None, **off)


def test_attention_that_is_not_causal_is_refused():
    for ways in (dict(is_causal=False), dict(module=dict(is_causal=False)), dict(module=dict(is_causal=False), is_causal=None)):
        with pytest.raises(ValueError, match="causal"):
            _Model(1)(4, None, **ways)
        _Model(1)(4, _mask([0], 0, 4), **ways)             # (the mask says what is seen)
        m = _Model(1)
        m(4, None)
        m(1, None, **ways)                                 # one token sees everything either way


@pytest.mark.parametrize("eight_bit", [True, False])
def test_tokens_beyond_the_capacity_are_refused(eight_bit):
    m = _Model(2, eight_bit=eight_bit)
    m(250, None)
    m(6, _mask([0, 0], 250, 6))
    for T in (1, 3):
        with pytest.raises(ValueError, match="capacity"):
            m(T, None)
    m.cache.reset()
    with pytest.raises(ValueError, match="capacity"):
        m(257, None)
