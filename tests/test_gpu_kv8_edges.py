"""8-bit KV pages on the GPU: calls at the edges of what their descriptions allow."""
import pytest
import torch

import kv8_ref as R
from test_gpu_kv8 import DEV, _check, _filled, _gen, _ints, _rand

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ waits
@pytest.mark.parametrize("D", [64, 128])
def test_row_tiles_of_a_chunk_start_one_after_the_other(D):
    """two full row tiles per CTA and many key tiles, over and over, beside other work on the same SMs: every wait ends and every bit
    is the same"""
    gen = _gen(D)
    n = 1500
    store, table, seqs = _filled(gen, [n], 2, D)
    q = _rand(gen, n, 8, D).to(DEV)
    call = lambda: store.chunk_attention(q, _ints([0, n]), table, _ints([n]), 0.1)            # noqa: E731
    want = call()
    rows = [0, 31, 63, 64, 127, 128, 700, n - 1]          # (of both row tiles of a CTA: 64 tokens are 256 rows)
    for i in rows:
        _check(want[i:i + 1], q[i:i + 1], [tuple(t[:i + 1] for t in seqs[0])], [0, 1], [i + 1], 0.1)
    torch.cuda.synchronize()
    side, other = torch.cuda.Stream(), torch.zeros(1 << 22, device=DEV)
    for _ in range(25):
        with torch.cuda.stream(side):
            other.mul_(0.5).add_(1.0)
        assert torch.equal(call(), want)
    torch.cuda.synchronize()
    from statetree_b200.ops import device_status
    assert device_status() == 0


# ------------------------------------------------------------------------------------------------ masks
@pytest.mark.parametrize("size,q_size,scale", [(0.0, 1e-30, 0.1), (0.0, 1e-38, 0.1), (1.0, 1.0, 1e-44), (0.0, 1.0, 1e-40)])
@pytest.mark.parametrize("D", [64, 128])
def test_masked_scores_whose_factor_is_below_fp32(D, size, q_size, scale):
    """the product of softmax scale, a page's key exponent and a query's is 0 in fp32: hidden keys still take no part"""
    gen = _gen(D)
    lens, new = [200, 77, 300], [200, 40, 300]
    store, table, seqs = _filled(gen, lens, 1, D, size=size)
    cu = [0, 200, 240, 540]
    q = (torch.randn(540, 4, D, generator=gen) * q_size).to(torch.bfloat16).to(DEV)
    for window, starts in ((0, None), (50, [0, 60, 131])):
        kw = dict(starts=None if starts is None else _ints(starts), window=window)
        got = store.chunk_attention(q, _ints(cu), table, _ints(lens), scale, **kw)
        _check(got, q, seqs, cu, lens, scale, starts, window)
        got = store.attention(q[:3], table, _ints(lens), scale, **kw)
        _check(got, q[:3], seqs, [0, 1, 2, 3], lens, scale, starts, window)


# ------------------------------------------------------------------------------------------------ block tables
def _both(store, q, table, lens, cu, **kw):
    n = table.shape[0]
    return store.attention(q[:n], table, lens, 0.1, **kw), store.chunk_attention(q, cu, table, lens, 0.1, **kw)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("rows", [20, 300])
def test_block_table_of_any_strides(native, rows, monkeypatch):
    """one row whose stride is not its width, part of a wider table, one row for all sequences: the same bits"""
    from statetree_b200 import kvcache
    gen = _gen(rows)
    store, table, _ = _filled(gen, [400], 2, 128)
    if not native:
        monkeypatch.setattr(kvcache, "calls", lambda: None)
    q = _rand(gen, rows, 8, 128).to(DEV)
    lens, cu = _ints([400]), _ints([0, rows])
    want = _both(store, q, table, lens, cu)
    line = table[0][:, None].t()
    assert line.shape == table.shape and line.stride() == (1, 1)
    wide = torch.cat([table + 1, table, table + 2], 1)[:, table.shape[1]:2 * table.shape[1]]
    for other in (line, wide, table.as_strided(table.shape, (3, 1))):
        for a, b in zip(want, _both(store, q, other, lens, cu)):
            assert torch.equal(a, b)
    lens, cu = _ints([400, 350, 20]), _ints([0, rows // 2, rows // 2, rows])
    want = _both(store, q, table.repeat(3, 1), lens, cu)
    for a, b in zip(want, _both(store, q, table.expand(3, -1), lens, cu)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("native", [True, False])
@pytest.mark.parametrize("rows", [20, 300])
def test_tokens_beyond_the_block_table(native, rows, monkeypatch):
    """lengths that the table has no pages for: what lies behind a row of it, in a wider table or behind its end, is not looked at"""
    from statetree_b200 import kvcache
    gen = _gen(rows)
    store, table, seqs = _filled(gen, [400, 400], 2, 128, table_extra=0)
    if not native:
        monkeypatch.setattr(kvcache, "calls", lambda: None)
    w = table.shape[1]
    wide = torch.cat([table.flip(1), table], 1)[:, w:]
    q = _rand(gen, rows, 8, 128).to(DEV)
    new = [0, rows // 2, rows]
    for splits in (1, 3):
        for lens in ([430, 500], [401, 400 + rows]):
            want, got = (_both(store, q, t, _ints(lens), _ints(new), splits=splits) for t in (table, wide))
            assert all(torch.equal(a, b) for a, b in zip(want, got))
            _check(got[0], q[:2], seqs, [0, 1, 2], lens, 0.1)
            _check(got[1], q, seqs, new, lens, 0.1)


# ------------------------------------------------------------------------------------------------ Hugging Face cache
@pytest.mark.parametrize("windows", [None, ["sliding_attention", "full_attention"], ["full_attention", "sliding_attention"]])
def test_hf_cache_with_padding_longer_than_a_chunk(windows):
    """a sequence behind 32 tokens of padding, in chunks of 16, against the same sequence by itself.  Both pass about twenty roundings
    to BF16 in two layers (2^-8 each: 7.8e-2 at most); the pages and their exponents are the same"""
    pytest.importorskip("transformers")
    from transformers import Qwen3Config, Qwen3ForCausalLM
    from statetree_b200.kvcache import StateTreeKVCache, enable
    cfg = Qwen3Config(vocab_size=512, hidden_size=256, intermediate_size=512, num_hidden_layers=2, num_attention_heads=4,
                      num_key_value_heads=2, head_dim=128, max_position_embeddings=256, tie_word_embeddings=False,
                      **(dict(use_sliding_window=True, sliding_window=8, layer_types=windows) if windows else {}))
    torch.manual_seed(0)
    model = enable(Qwen3ForCausalLM(cfg).to(torch.bfloat16).cuda().eval())
    P, pad, ends = 50, 32, [16, 32, 48, 50, 51, 52]
    ids = torch.randint(0, cfg.vocab_size, (2, 52), device="cuda")
    mask = torch.ones(2, 52, dtype=torch.long, device="cuda")
    mask[1, :pad] = 0
    at = torch.arange(52, device="cuda").repeat(2, 1)
    at[1] = (at[1] - pad).clamp(min=0)

    def passes(rows, first, ends):
        cache, outs = StateTreeKVCache(model.config, batch_size=len(rows), max_cache_len=64, eight_bit=True), []
        with torch.no_grad():
            for a, b in zip([first] + ends, ends):
                outs.append(model(input_ids=ids[rows, a:b], attention_mask=mask[rows, first:b], position_ids=at[rows, a:b],
                                  past_key_values=cache, use_cache=True).logits[:, -1].float())
        cache.check()
        return outs

    both = passes([0, 1], 0, ends)
    for row, first in ((0, 0), (1, pad)):
        for got, want in zip(both[2:], passes([row], first, [48, 50, 51, 52])):
            assert float((got[row] - want[0]).norm() / want[0].norm()) < 2 * 20 * 2.0 ** -8, (row, first)


def test_hf_cache_masks_in_a_captured_pass():
    """a captured chunk reads its mask's padding when it is replayed; a mask that an eager pass refuses shows in check()"""
    pytest.importorskip("transformers")
    import types
    from statetree_b200.kvcache import StateTreeKVCache, statetree_attention
    B, T = 2, 24
    cfg = types.SimpleNamespace(num_hidden_layers=2, num_attention_heads=4, num_key_value_heads=2)
    cache = StateTreeKVCache(cfg, batch_size=B, max_cache_len=64, eight_bit=True)
    gen = _gen(1)
    q, k, v = (_rand(gen, B, h, T, 128).to(DEV) for h in (4, 2, 2))
    at = torch.arange(T, device=DEV)
    plain = lambda pads: ((at <= at[:, None]) & (at >= _ints(pads)[:, None, None]))[:, None]  # noqa: E731
    mask = plain([0, 0])

    def step():
        outs = []
        for i in range(2):
            cache.update(k, v, i)
            outs.append(statetree_attention(types.SimpleNamespace(layer_idx=i), q, k, v, mask, scaling=0.1)[0])
        return outs

    step()
    cache.reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for pads in ([0, 5], [3, 0]):
        mask.copy_(plain(pads))
        cache.reset()
        graph.replay()
        got = [o.clone() for o in outs]
        cache.check()
        cache.reset()
        assert all(torch.equal(a, b) for a, b in zip(got, step()))
    mask[0, 0, 20, 7] = False                              # one hidden key
    cache.reset()
    graph.replay()
    with pytest.raises(ValueError, match="mask"):
        cache.check()
    cache.reset()
    cache.check()
    with pytest.raises(ValueError, match="mask"):
        step()


# ------------------------------------------------------------------------------------------------ precision
def _close(q, seqs, cu, lens, scale, got):
    """the kernels' own bound, per value: probabilities rounded to FP16 (2^-11 of each at most, or, where that is subnormal, 2^-32 of the
    largest times its page's largest value, at most twice the largest of all values), the output rounded to BF16 (2^-8), scores summed
    in fp32 over D products (each sum off by at most D 2^-24 of its absolute sum, twice since the reference is subtracted; the factors
    and the difference four roundings more), sums over the keys (2^-24 each), the exponential (2^-21 with its argument's rounding)"""
    got = got.cpu().double()
    for b, (K, V) in enumerate(seqs):
        n, L, D = cu[b + 1] - cu[b], lens[b], q.shape[-1]
        out, mag, wide = R.attend(q[cu[b]:cu[b + 1]].cpu().double(), K, V, list(range(L - n, L)), scale)
        rel = 2.0 ** -11 + 2 * (D + 4) * 2.0 ** -24 * wide[..., None] + L * 2.0 ** -24 + 2.0 ** -21
        near = mag * rel * 1.01 + L * 2.0 ** -31 * float(V.abs().max())
        off = (got[cu[b]:cu[b + 1]] - out).abs()
        assert bool((off <= near + 2.0 ** -8 * (out.abs() + near)).all()), (b, float((off / (near + 2.0 ** -8 * out.abs())).max()))


def _opposed(gen, n, H, D, spread):
    """keys of which two share the weight almost evenly, their values opposed, the others far below: the output is a difference of two
    probabilities, in which a rounding of either shows"""
    K, V = torch.zeros(n, H, D), torch.zeros(n, H, D)
    K[:, :, 0] = -24.0
    K[:2, :, 0] = 0.0
    K[:2, :, 1:9] = torch.randn(2, H, 8, generator=gen) * spread
    V[0], V[1] = 1.0, -1.0
    V[2:] = torch.randn(n - 2, H, D, generator=gen)
    return K, V


@pytest.mark.parametrize("D,H,G", [(128, 2, 4), (64, 1, 7)])
@pytest.mark.parametrize("spread", [0.02, 0.2])
def test_probabilities_have_eleven_bits(D, H, G, spread):
    gen = _gen(D)
    n, new = 150, 70
    store, table, _ = _filled(gen, [n], H, D)
    K, V = _opposed(gen, n, H, D, spread)
    p = torch.arange(n)
    store.append(K.to(torch.bfloat16).to(DEV), V.to(torch.bfloat16).to(DEV), (table[0].cpu()[p // 16] * 16 + p % 16).to(DEV))
    seqs = [tuple(t.cpu().double().flatten(0, 1)[:n] for t in store.dense(table[0, :-(-n // 16)].contiguous()))]
    q = torch.randn(new, H * G, D, generator=gen)
    q[:, :, 0] = 1.0
    q = q.to(torch.bfloat16).to(DEV)
    for rows, splits in ((1, 1), (1, 3), (4, 1), (4, 2), (new, 1), (new, 2)):
        got = store.chunk_attention(q[:rows], _ints([0, rows]), table, _ints([n]), 1.0, splits=splits)
        _close(q[:rows], seqs, [0, rows], [n], 1.0, got)
    _close(q[:1], seqs, [0, 1], [n], 1.0, store.attention(q[:1], table, _ints([n]), 1.0, splits=2, min_pages=1))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("splits", [1, 3, 11])
def test_precision_of_random_scores(D, splits):
    gen = _gen(splits)
    lens, cu = [300, 33, 700], [0, 60, 63, 200]
    store, table, seqs = _filled(gen, lens, 2, D)
    q = _rand(gen, 200, 8, D, size=1.5).to(DEV)
    _close(q, seqs, cu, lens, D ** -0.5, store.chunk_attention(q, _ints(cu), table, _ints(lens), D ** -0.5, splits=splits))
    got = store.attention(q[:3], table, _ints(lens), D ** -0.5, splits=splits, min_pages=1)
    _close(q[:3], seqs, [0, 1, 2, 3], lens, D ** -0.5, got)
    few = [0, 4, 5, 9]
    got = store.chunk_attention(q[:9], _ints(few), table, _ints(lens), D ** -0.5, splits=splits)
    _close(q[:9], seqs, few, lens, D ** -0.5, got)


# ------------------------------------------------------------------------------------------------ refusals
def test_both_host_paths_refuse_the_same(monkeypatch):
    """what a call of wrong form is told does not depend on the native host path"""
    from statetree_b200 import kvcache
    store = kvcache.PageStore8(4, 2, DEV)
    bf = lambda *s: torch.zeros(*s, dtype=torch.bfloat16, device=DEV)                         # noqa: E731
    f32 = lambda *s: torch.zeros(*s, device=DEV)                                              # noqa: E731
    K, slots = bf(3, 2, 128), torch.zeros(3, dtype=torch.int64, device=DEV)
    table, lens, q = torch.zeros(3, 4, dtype=torch.int32, device=DEV), _ints([0, 0, 0]), bf(3, 4, 128)
    calls = [(store.append, dict(K=K, V=K, slots=slots), bad) for bad in (
        dict(K=bf(3, 2, 64)), dict(K=bf(3, 1, 128), V=bf(3, 1, 128)), dict(V=bf(2, 2, 128)), dict(K=f32(3, 2, 128)), dict(slots=slots[:2]),
        dict(slots=slots.int()), dict(slots=slots.cpu()), dict(V=K.cpu()), dict(cos=f32(9, 64)), dict(cos=f32(9, 64), sin=f32(9, 64)),
        dict(cos=f32(9, 32), sin=f32(9, 32), positions=slots), dict(cos=f32(9, 64), sin=f32(9, 64), positions=slots[:2]),
        dict(k_norm=bf(64)), dict(q=bf(2, 4, 128)), dict(q=q, q_out=bf(3, 5, 128)), dict(q=q, q_out=bf(3, 1, 128).expand(3, 4, 128)))]
    one = dict(q=q, block_table=table, lens=lens, scale=0.1)
    calls += [(store.attention, one, bad) for bad in (
        dict(q=bf(3, 3, 128)), dict(q=bf(2, 4, 128)), dict(lens=lens.long()), dict(lens=lens[:2]), dict(block_table=table.long()),
        dict(block_table=table[:, :0]), dict(block_table=table.repeat(1, 2)[:, ::2]), dict(starts=lens[:1]), dict(window=-1), dict(splits=0),
        dict(out=bf(3, 2, 128)), dict(q=q.float()), dict(scale=0.0), dict(scale=float("nan")), dict(splits=2000), dict(lens=lens.cpu()))]
    calls += [(store.chunk_attention, dict(one, cu=_ints([0, 1, 2, 3])), bad) for bad in (
        dict(cu=lens), dict(cu=_ints([0, 1, 2, 3]).long()), dict(cu=None, q=bf(5, 4, 128)), dict(splits=0), dict(window=-1))]
    said = []
    for native in (True, False):
        if not native:
            monkeypatch.setattr(kvcache, "calls", lambda: None)
        said.append([])
        for call, good, bad in calls:
            with pytest.raises(RuntimeError) as e:
                call(**{**good, **bad})
            said[-1].append(str(e.value))
    assert said[0] == said[1]
    torch.cuda.synchronize()


# ------------------------------------------------------------------------------------------------ scores beyond fp32
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("splits", [1, 2, 3])
def test_scores_below_fp32(D, splits):
    """finite queries and keys whose product no fp32 number holds, far below all others: those keys weigh nothing, wherever they stand"""
    gen = _gen(D)
    n, H = 200, 1
    store, table, _ = _filled(gen, [n], H, D)
    for lows in ([0], [0, 1, 2], [3], [2, 12], list(range(12))):                             # pages of such keys
        K, V = torch.zeros(n, H, D), _rand(gen, n, H, D)
        for p in lows:
            K[p * 16:(p + 1) * 16] = -1e3
        at = torch.arange(n)
        slots = table[0].cpu()[at // 16] * 16 + at % 16
        store.append(K.to(torch.bfloat16).to(DEV), V.to(DEV), slots.to(DEV))
        seqs = [tuple(t.cpu().double().flatten(0, 1)[:n] for t in store.dense(table[0, :-(-n // 16)].contiguous()))]
        q = torch.full((80, 4, D), 3e38, dtype=torch.bfloat16, device=DEV)
        _check(store.attention(q[:1], table, _ints([n]), 0.1, splits=splits, min_pages=1), q[:1], seqs, [0, 1], [n], 0.1)
        for rows in (1, 3, 80):
            # (rows all of whose keys are such: no answer in fp32)
            rows = min(rows, n - 16 * (max(lows) + 1) + 16) if len(lows) < 12 else 1
            got = store.chunk_attention(q[:rows], _ints([0, rows]), table, _ints([n]), 0.1, splits=splits)
            _check(got, q[:rows], seqs, [0, rows], [n], 0.1)


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("splits", [1, 3, 12])
def test_queries_that_are_no_numbers(splits, bad):
    """give outputs that are none, and leave every other row and head as it is"""
    gen = _gen(splits)
    lens, H = [300, 70, 0], 2
    store, table, _ = _filled(gen, lens, H, 128)
    for cu in (None, [0, 5, 8, 8], [0, 200, 270, 270]):
        q = _rand(gen, cu[-1] if cu else 3, 8, 128).to(DEV)
        call = lambda q: (store.attention(q, table, _ints(lens), 0.1, splits=splits, min_pages=1) if cu is None else      # noqa: E731
                          store.chunk_attention(q, _ints(cu), table, _ints(lens), 0.1, splits=splits))
        want = call(q)
        q[1, 5, 17] = bad
        got = call(q)
        assert bool(got[1, 5].isnan().all())
        got[1, 5] = want[1, 5]
        assert torch.equal(got, want)
