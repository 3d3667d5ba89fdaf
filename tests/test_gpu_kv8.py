"""8-bit KV pages on the GPU against their plain 64-bit statement (kv8_ref): append with and without rotation, read-back, attention of
one and of several query tokens per sequence."""
import pytest
import torch

import kv8_ref as R

pytestmark = pytest.mark.gpu
DEV = "cuda"
PAGE = 16


def _store(blocks, H, D):
    from statetree_b200.kvcache import PageStore8
    return PageStore8(blocks, H, DEV, head_dim=D)


def _rand(gen, *shape, size=1.0):
    return (torch.randn(*shape, generator=gen) * size).to(torch.bfloat16)


def _keys(gen, n, H, D):
    return (torch.randn(n, H, D, generator=gen) * torch.randn(H, D, generator=gen).exp()).to(torch.bfloat16)


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _same(store, ref):
    """every stored value and exponent equals the statement's"""
    for got, want in zip(store.dense(), ref.dense()):
        assert torch.equal(got.cpu().double(), want)
    assert torch.equal(store.exps.cpu().long(), ref.exps)
    assert int(store.marks.abs().max()) == 0


# ------------------------------------------------------------------------------------------------ append
@pytest.mark.parametrize("D,H", [(128, 1), (128, 8), (64, 3)])
@pytest.mark.parametrize("calls", [(1,), (16,), (5, 1, 1, 20, 3), (40, 600, 1, 7), (385,), (2401,)])
def test_append_in_order(D, H, calls):
    """a sequence that grows over several calls (whole pages, parts of pages, single tokens; short and long calls)"""
    gen = _gen(sum(calls) + D + H)
    blocks = -(-sum(calls) // PAGE) + 3
    store, ref = _store(blocks, H, D), R.Pages(blocks, H, D)
    order, at = torch.randperm(blocks, generator=gen), 0
    for n in calls:
        K, V = _keys(gen, n, H, D), _rand(gen, n, H, D, size=10.0 ** torch.randint(-3, 4, (1,), generator=gen).item())
        p = torch.arange(at, at + n)
        slots = order[p // PAGE] * PAGE + p % PAGE
        store.append(K.to(DEV), V.to(DEV), slots.to(DEV))
        ref.append(K.double(), V.double(), slots)
        at += n
    _same(store, ref)
    store.check()
    some = torch.tensor([blocks - 1, 0, 0, blocks, -1], device=DEV)
    for got, want in zip(store.dense(some), ref.dense()):
        assert torch.equal(got.cpu().double()[:3], want[[blocks - 1, 0, 0]]) and not got[3:].any()


@pytest.mark.parametrize("n", [1, 33, 384, 385, 700, 2500])
def test_append_any_order(n):
    """slots in any order, padding and slots beyond the cache, the same slot several times (the last token counts), pages that do
    not start anew and pages that do"""
    H, D, blocks = 2, 128, 30
    gen = _gen(n)
    store, ref = _store(blocks, H, D), R.Pages(blocks, H, D)
    for size in (1.0, 30.0, 0.01):
        K, V = _keys(gen, n, H, D), _rand(gen, n, H, D, size=size)
        slots = torch.randint(-20, (blocks + 2) * PAGE, (n,), generator=gen)
        store.append(K.to(DEV), V.to(DEV), slots.to(DEV))
        ref.append(K.double(), V.double(), slots)
        _same(store, ref)


def test_append_single_tokens_raise_the_exponent():
    """a page filled token by token by ever larger values: its old rows are rounded again, and no other page is touched"""
    H, D = 3, 64
    gen = _gen(5)
    store, ref = _store(4, H, D), R.Pages(4, H, D)
    store.pages.fill_(0x3C)
    store.exps.fill_(3)
    untouched = store.pages.clone()
    for r in range(PAGE):
        K, V = _rand(gen, 1, H, D, size=2.0 ** (r - 4)), _rand(gen, 1, H, D, size=4.0 ** (8 - r))
        slots = torch.tensor([2 * PAGE + r])
        store.append(K.to(DEV), V.to(DEV), slots.to(DEV))
        ref.append(K.double(), V.double(), slots)
        assert torch.equal(store.dense(torch.tensor([2], device=DEV))[0].cpu().double(), ref.dense()[0][2:3])
        assert torch.equal(store.dense(torch.tensor([2], device=DEV))[1].cpu().double(), ref.dense()[1][2:3])
    for p in (0, 1, 3):
        assert torch.equal(store.pages[p], untouched[p]) and bool((store.exps[p] == 3).all())


def test_append_extremes():
    """zeros, the smallest and largest values, borders of the exponent (448 * 2^e and the next BF16 number), ties of the rounding"""
    H, D = 1, 64
    rows = [torch.zeros(D), torch.full((D,), 448.0), torch.full((D,), 450.0), torch.full((D,), 7.0), torch.full((D,), 7.03125),
            torch.full((D,), 1e-20), torch.full((D,), 3e19), torch.linspace(0, 2, D), torch.full((D,), 1e-40),
            torch.arange(D) * 2.0 ** -10 + 448 * (torch.arange(D) == 0), torch.tensor([17.0, 19.0, 21.0, 23.0] * 16)]
    for size in rows:
        store, ref = _store(1, H, D), R.Pages(1, H, D)
        x = torch.stack([size, -size]).to(torch.bfloat16)[:, None]
        slots = torch.tensor([0, 1])
        store.append(x.to(DEV), x.to(DEV), slots.to(DEV))
        ref.append(x.double(), x.double(), slots)
        _same(store, ref)
        store.check()


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_append_what_the_format_cannot_hold(bad):
    store, ref = _store(2, 2, 64), R.Pages(2, 2, 64)
    x = _rand(_gen(1), 20, 2, 64)
    x[7, 1, 5] = bad
    slots = torch.arange(20)
    store.append(x.to(DEV), x.to(DEV), slots.to(DEV))
    y = x.double()
    if abs(bad) == float("inf"):                          # the largest of the block's exponent
        y[7, 1, 5] = 0
        e = R.exponent(float(y[:16, 1].abs().max()))
        y[7, 1, 5] = 448 * 2.0 ** e * (1 if bad > 0 else -1)
    ref.append(y, y, slots)
    _same(store, ref)
    with pytest.raises(RuntimeError, match="finite"):
        store.check()
    store.reset()
    store.check()


def test_append_what_the_format_cannot_hold_in_long_calls():
    """the same in many pages of one call, in either half of them, beside the largest value and away from it"""
    H, D, n = 3, 128, 500
    store, ref = _store(33, H, D), R.Pages(33, H, D)
    gen = _gen(2)
    K, V = _keys(gen, n, H, D), _rand(gen, n, H, D)
    y, inf = [], float("inf")
    for X in (K, V):
        at = torch.randint(0, n, (40,), generator=gen), torch.randint(0, H, (40,), generator=gen), torch.randint(0, D, (40,), generator=gen)
        X[at] = torch.tensor([float("nan"), inf, -inf, 3e38])[torch.arange(40) % 4].to(torch.bfloat16)
        Y = X.double()
        for p in range(0, n, PAGE):                       # infinities: the largest of the block's exponent
            for h in range(H):
                block = Y[p:p + PAGE, h]
                fine = torch.where(block.isfinite(), block, torch.zeros_like(block))
                top = 448 * 2.0 ** R.exponent(float(fine.abs().max()))
                Y[p:p + PAGE, h] = torch.where(block.isnan(), torch.zeros_like(block), block.clamp(-top, top))
        y.append(Y)
    slots = torch.arange(n) + PAGE
    store.append(K.to(DEV), V.to(DEV), slots.to(DEV))
    ref.append(y[0], y[1], slots)
    _same(store, ref)
    with pytest.raises(RuntimeError, match="finite"):
        store.check()


@pytest.mark.parametrize("n", [1, 400])
def test_append_without_an_epsilon(n):
    """norms with eps = 0: rows of a page that no token goes to are not taken for values (0 * rsqrt(0) is not a number)"""
    H, D = 2, 128
    gen = _gen(n)
    K, V = _keys(gen, n, H, D), _rand(gen, n, H, D)
    w = (1 + 0.1 * torch.randn(D, generator=gen)).to(torch.bfloat16)
    slots = torch.arange(n) + 2
    store, other = _store(n // PAGE + 2, H, D), _store(n // PAGE + 2, H, D)
    store.append(K.to(DEV), V.to(DEV), slots.to(DEV), k_norm=w.to(DEV), eps=0.0)
    store.check()
    other.append(K.to(DEV), V.to(DEV), slots.to(DEV), k_norm=w.to(DEV), eps=1e-30)       # (the same sum in fp32)
    assert torch.equal(store.pages, other.pages) and torch.equal(store.exps, other.exps)
    K[0, 1] = 0                                            # a token that is zero has no norm
    store.append(K.to(DEV), V.to(DEV), slots.to(DEV), k_norm=w.to(DEV), eps=0.0)
    with pytest.raises(RuntimeError, match="not finite"):
        store.check()


def _tables(D, span):
    inv = 1e6 ** (-torch.arange(0, D, 2, dtype=torch.float64) / D)
    ang = torch.arange(span, dtype=torch.float64)[:, None] * inv
    return ang.cos().float(), ang.sin().float()


@pytest.mark.parametrize("interleaved", [True, False])
@pytest.mark.parametrize("D,H,Hq,n,normed", [(128, 8, 32, 3, True), (64, 2, 14, 70, False), (128, 1, 5, 600, True), (64, 3, 3, 530, True), (128, 2, 2, 1, False)])
def test_append_rotates(interleaved, D, H, Hq, n, normed):
    """keys and queries of a fused projection's rows, normalised and rotated at positions of their own"""
    gen = _gen(n + D)
    blocks, span = -(-n // PAGE) + 1, 900
    cos, sin = _tables(D, span)
    wide = torch.cat([_rand(gen, n, Hq, D), _keys(gen, n, H, D), _rand(gen, n, H, D)], 1).flatten(1)
    q, k, v = wide.to(DEV).view(n, Hq + 2 * H, D).split([Hq, H, H], 1)
    pos = torch.randint(-3, span + 5, (n,), generator=gen)
    wq, wk = (1 + 0.2 * torch.randn(2, D, generator=gen)).to(torch.bfloat16)
    wq, wk = (wq, wk) if normed else (None, None)
    slots = torch.arange(n) + 3
    store = _store(blocks, H, D)
    to = lambda t: None if t is None else t.to(DEV)                                           # noqa: E731
    out = store.append(k, v, slots.to(DEV), positions=pos.to(DEV), cos=to(cos), sin=to(sin), interleaved=interleaved, q=q, q_norm=to(wq),
                       k_norm=to(wk), eps=1e-5)
    at = pos.clamp(0, span - 1)
    c, s = cos[at][:, None], sin[at][:, None]

    def exact(x, w):
        x = x.cpu().double()
        y = x if w is None else R.norm(x, w, 1e-5)
        # a rotated value is off by the roundings of two products and a sum, of the norm by those of its sum, its root (2^-22) and two
        # products: together below 2^-19 of what the pair holds
        pair = R.rotate(y.abs(), torch.ones_like(c), torch.ones_like(s), interleaved).abs() + y.abs()
        return R.rotate(y, c, s, interleaved), pair * 2.0 ** -19

    y, tol = exact(q, wq)
    assert bool(((out.cpu().double() - y).abs() <= tol + 2.0 ** -8 * y.abs()).all())
    y, tol = exact(k, wk)
    kd, vd = store.dense()
    ref = R.Pages(blocks, H, D)
    ref.append(v.cpu().double(), v.cpu().double(), slots)
    assert torch.equal(vd.cpu().double(), ref.dense()[1])
    got = kd.cpu().double().flatten(0, 1)[3:3 + n]
    e = store.exps[:, :, 0].cpu().double().repeat_interleave(PAGE, 0)[3:3 + n][..., None]
    assert bool(((got - y).abs() <= tol + torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** (e - 10))).all())
    for p in range(blocks):                               # the exponent is the block's (of values that far from exact)
        mine = (slots // PAGE == p).nonzero()[:, 0]
        for h in range(H):
            if len(mine):
                top = y[mine, h].abs().max()
                assert R.exponent(float(top * (1 - 2e-6))) <= int(store.exps[p, h, 0]) <= R.exponent(float(top * (1 + 2e-6)))


def test_append_one_position_for_all_and_in_place():
    D, H = 128, 2
    gen = _gen(9)
    cos, sin = (t.to(DEV) for t in _tables(D, 50))
    k, v, q = (_rand(gen, 4, H, D).to(DEV) for _ in range(3))
    slots = torch.tensor([0, 17, 40, -1], device=DEV)
    a, b = _store(4, H, D), _store(4, H, D)
    out = a.append(k, v, slots, positions=torch.tensor([31], device=DEV), cos=cos, sin=sin, q=q)
    mine = q.clone()
    same = b.append(k, v, slots, positions=torch.full((4,), 31, device=DEV), cos=cos, sin=sin, q=mine, q_out=mine)
    assert same is mine and torch.equal(out, mine) and torch.equal(a.pages, b.pages) and torch.equal(a.exps, b.exps)


def test_append_other_layouts():
    """heads not contiguous, odd strides, an unaligned start, one token for all rows: copied as needed, the same pages"""
    D, H, n = 64, 3, 21
    gen = _gen(3)
    K, V = _rand(gen, n, H, D).to(DEV), _rand(gen, n, H, D).to(DEV)
    slots = torch.arange(n, device=DEV)
    want = _store(2, H, D)
    want.append(K, V, slots)
    odd = torch.zeros(n * H * D + 3, dtype=torch.bfloat16, device=DEV)[3:].view(n, H, D).copy_(V)
    other = _store(2, H, D)
    other.append(K.transpose(0, 1).contiguous().transpose(0, 1), odd, slots)
    assert torch.equal(other.pages, want.pages) and torch.equal(other.exps, want.exps)
    wide = torch.zeros(n, H * D + 4, dtype=torch.bfloat16, device=DEV)
    wide[:, :H * D] = K.flatten(1)
    other = _store(2, H, D)
    other.append(wide[:, :H * D].view(n, H, D), V, slots)
    assert torch.equal(other.pages, want.pages)
    one, two = _store(2, H, D), _store(2, H, D)
    one.append(K[:1].expand(n, H, D), V[:1].expand(n, H, D), slots)
    two.append(K[:1].repeat(n, 1, 1), V[:1].repeat(n, 1, 1), slots)
    assert torch.equal(one.pages, two.pages)


# ------------------------------------------------------------------------------------------------ attention
def _filled(gen, lens, H, D, spare=3, size=1.0, table_extra=2):
    """(store, block table, [(K, V) float64 of each sequence]): pages in any order; pages of no sequence, rows behind a sequence's
    last token and table entries behind its last page hold what must not be read"""
    per = [-(-n // PAGE) for n in lens]
    blocks = sum(per) + spare
    store = _store(blocks, H, D)
    store.pages.copy_(torch.randint(0, 256, store.pages.shape, generator=gen).to(torch.uint8))
    store.exps.fill_(56)
    order = torch.randperm(blocks, generator=gen)
    width = max(1, max(per)) + table_extra
    table = torch.randint(-5, blocks + 5, (len(lens), width), generator=gen)
    seqs, at = [], 0
    for b, n in enumerate(lens):
        table[b, :per[b]] = order[at:at + per[b]]
        at += per[b]
        K, V = _keys(gen, n, H, D) * size, _rand(gen, n, H, D, size=3.0)
        if n:
            p = torch.arange(n)
            store.append(K.to(torch.bfloat16).to(DEV), V.to(DEV), (table[b][p // PAGE] * PAGE + p % PAGE).to(DEV))
        mine = table[b, :per[b]].to(DEV)
        if n % PAGE:                                      # rows behind the last token
            store.pages[mine[-1], :, :, n % PAGE:] = 0x7E
        kd, vd = store.dense(mine) if n else (torch.zeros(0, PAGE, H, D),) * 2
        seqs.append((kd.cpu().double().flatten(0, 1)[:n], vd.cpu().double().flatten(0, 1)[:n]))
    return store, table.to(torch.int32).to(DEV), seqs


def _check(got, q, seqs, cu, lens, scale, starts=None, window=0):
    got = got.cpu().double()
    for b, (K, V) in enumerate(seqs):
        n = cu[b + 1] - cu[b]
        if n == 0:
            continue
        pos = list(range(lens[b] - n, lens[b]))
        out, mag, wide = R.attend(q[cu[b]:cu[b + 1]].cpu().double(), K, V, pos, scale, starts[b] if starts else 0, window)
        off = (got[cu[b]:cu[b + 1]] - out).abs()
        tol = R.allowed(out, mag, wide, max(lens[b], 1), q.shape[-1])
        assert bool((off <= tol).all()), (b, float((off / tol).max()), [int(x) for x in (off > tol).nonzero()[0]])


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("D,H,G", [(128, 8, 4), (128, 2, 1), (128, 1, 8), (64, 2, 7), (64, 3, 3), (128, 1, 16), (64, 1, 20)])
@pytest.mark.parametrize("splits", [1, 3, 8, 12, None])
def test_decode_attention(D, H, G, splits):
    lens = [1, 0, 15, 16, 17, 33, 130, 700]
    gen = _gen(D + H + G)
    store, table, seqs = _filled(gen, lens, H, D)
    q = _rand(gen, len(lens), H * G, D, size=1.5).to(DEV)
    got = store.attention(q, table, _ints(lens), D ** -0.5, splits=splits, min_pages=1)
    assert not got[1].any()                               # a sequence without tokens
    _check(got, q, seqs, list(range(len(lens) + 1)), lens, D ** -0.5)
    assert torch.equal(got, store.attention(q, table, _ints(lens), D ** -0.5, splits=splits, min_pages=1))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("window", [0, 1, 5, 64, 1000])
@pytest.mark.parametrize("splits", [1, 4, 11])
def test_decode_attention_masks(D, window, splits):
    """left padding (up to the whole sequence and beyond) and sliding windows"""
    lens, starts = [40, 40, 40, 40, 333, 333, 16], [0, 7, 39, 40, 100, 16, 50]
    gen = _gen(D + window)
    store, table, seqs = _filled(gen, lens, 2, D)
    q = _rand(gen, len(lens), 8, D).to(DEV)
    got = store.attention(q, table, _ints(lens), 0.2, splits=splits, starts=_ints(starts), window=window, min_pages=1)
    assert not got[3].any() and not got[6].any()
    _check(got, q, seqs, list(range(len(lens) + 1)), lens, 0.2, starts, window)


@pytest.mark.parametrize("size", [1e-3, 40.0])
def test_attention_of_flat_and_peaked_scores(size):
    """scores that are all alike, and scores hundreds apart (one key takes everything; maxima that rise along the sequence)"""
    gen = _gen(11)
    lens = [500, 77]
    store, table, seqs = _filled(gen, lens, 2, 128, size=size)
    q = _rand(gen, 2, 8, 128, size=4.0).to(DEV)
    _check(store.attention(q, table, _ints(lens), 0.09, splits=2, min_pages=1), q, seqs, [0, 1, 2], lens, 0.09)
    cu = [0, 130, 207]
    q = _rand(gen, 207, 8, 128, size=4.0).to(DEV)
    _check(store.chunk_attention(q, _ints(cu), table, _ints(lens), 0.09), q, seqs, cu, lens, 0.09)


def test_attention_of_small_and_large_values():
    """codes below the normal range of e4m3 and exponents far apart from page to page"""
    gen = _gen(4)
    H, D, n = 1, 64, 80
    store, table, _ = _filled(gen, [n], H, D)
    K, V = _rand(gen, n, H, D), _rand(gen, n, H, D)
    K *= torch.where(torch.rand(n, H, D, generator=gen) < 0.1, 1.0, 2.0 ** -9).to(torch.bfloat16)
    V *= torch.tensor([2.0 ** (12 * (i // PAGE) - 24) for i in range(n)])[:, None, None].to(torch.bfloat16)
    p = torch.arange(n)
    store.append(K.to(DEV), V.to(DEV), (table[0].cpu()[p // PAGE] * PAGE + p % PAGE).to(DEV))
    kd, vd = (t.cpu().double().flatten(0, 1)[:n] for t in store.dense(table[0, :5].contiguous()))
    q = _rand(gen, 20, 4, D, size=4.0).to(DEV)
    for at in (16, 33, 80):
        _check(store.attention(q[:1], table, _ints([at]), 0.3), q[:1], [(kd, vd)], [0, 1], [at], 0.3)
    _check(store.chunk_attention(q, _ints([0, 20]), table, _ints([n]), 0.3), q, [(kd, vd)], [0, 20], [n], 0.3)


CHUNKS = [([1], [1]), ([5], [5]), ([20], [3]), ([300], [300]), ([700], [129]), ([64, 0, 17, 500, 33, 16], [4, 0, 17, 250, 1, 0]),
          ([129, 260, 257], [129, 130, 257])]


@pytest.mark.parametrize("lens,new", CHUNKS)
@pytest.mark.parametrize("D,H,G", [(128, 2, 4), (64, 2, 7), (128, 1, 1), (64, 1, 16), (128, 3, 3)])
def test_chunk_attention(lens, new, D, H, G):
    gen = _gen(sum(lens) + D + G)
    store, table, seqs = _filled(gen, lens, H, D)
    cu = [sum(new[:b]) for b in range(len(new) + 1)]
    q = _rand(gen, cu[-1], H * G, D, size=1.5).to(DEV)
    got = store.chunk_attention(q, _ints(cu), table, _ints(lens), D ** -0.5)
    _check(got, q, seqs, cu, lens, D ** -0.5)
    assert torch.equal(got, store.chunk_attention(q, _ints(cu), table, _ints(lens), D ** -0.5))


@pytest.mark.parametrize("splits", [1, 2, 5])
@pytest.mark.parametrize("window", [0, 1, 40, 300])
@pytest.mark.parametrize("D", [64, 128])
def test_chunk_attention_masks(D, window, splits):
    """windows, left padding (rows that see nothing are zero), more queries than tokens, rows behind the last sequence"""
    lens, new, starts = [400, 30, 130, 7], [200, 30, 5, 12], [0, 11, 300, 2]
    gen = _gen(D + window)
    store, table, seqs = _filled(gen, lens, 2, D)
    cu = [sum(new[:b]) for b in range(len(new) + 1)]
    q = _rand(gen, cu[-1] + 9, 6, D).to(DEV)
    out = torch.full_like(q, 5.0)
    got = store.chunk_attention(q, _ints(cu), table, _ints(lens), 0.15, starts=_ints(starts), window=window, splits=splits, out=out)
    assert got is out and bool((out[cu[-1]:] == 5.0).all())
    _check(got, q, seqs, cu, lens, 0.15, starts, window)
    assert not got[cu[1]:cu[1] + 11].any() and not got[cu[2]:cu[3]].any() and not got[cu[3]:cu[3] + 5].any()


@pytest.mark.parametrize("splits", [1, 2, 7, 12])
@pytest.mark.parametrize("window", [0, 1, 40])
@pytest.mark.parametrize("D", [64, 128])
def test_attention_of_few_rows(D, window, splits):
    """chunks of a few tokens: as above, rows of one sequence that share a CTA with other tokens' and a sequence without queries"""
    lens, new, starts = [400, 30, 130, 3, 900], [4, 0, 1, 5, 7], [0, 11, 300, 1, 5]
    gen = _gen(D + window)
    store, table, seqs = _filled(gen, lens, 2, D)
    cu = [sum(new[:b]) for b in range(len(new) + 1)]
    q = _rand(gen, cu[-1] + 2, 6, D).to(DEV)
    out = torch.full_like(q, 5.0)
    got = store.chunk_attention(q, _ints(cu), table, _ints(lens), 0.15, starts=_ints(starts), window=window, splits=splits, out=out)
    assert bool((out[cu[-1]:] == 5.0).all())
    _check(got, q, seqs, cu, lens, 0.15, starts, window)
    assert not got[4].any() and not got[5:8].any()        # (all keys padding; positions -2, -1 and the padded 0)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("splits", [2, 5])
def test_attention_of_more_than_a_wave(D, splits):
    """so many sequences that their splits do not join on chip"""
    lens = [(37 * b) % 150 for b in range(90)]
    gen = _gen(D + splits)
    store, table, seqs = _filled(gen, lens, 8, D)
    q = _rand(gen, len(lens), 8, D).to(DEV)
    got = store.attention(q, table, _ints(lens), 0.1, splits=splits, min_pages=1)
    _check(got, q, seqs, list(range(len(lens) + 1)), lens, 0.1)
    cu = [min(2 * b, 120) for b in range(len(lens) + 1)]
    lens = [max(n, 2) for n in lens]
    q = _rand(gen, 120, 16, D).to(DEV)
    got = store.chunk_attention(q, _ints(cu), table, _ints(lens), 0.1, splits=splits)
    mine = [(K, V) if len(K) >= 2 else None for K, V in seqs]
    for b, s in enumerate(mine):
        if s is not None:
            _check(got[cu[b]:cu[b + 1]], q[cu[b]:cu[b + 1]], [s], [0, cu[b + 1] - cu[b]], [lens[b]], 0.1)


@pytest.mark.parametrize("splits", [1, 4, 12])
def test_attention_into_its_queries(splits):
    gen = _gen(splits)
    store, table, _ = _filled(gen, [300, 40], 2, 128)
    lens, cu = _ints([300, 40]), _ints([0, 3, 5])
    for n, call in ((2, lambda q, out: store.attention(q, table, lens, 0.1, splits=splits, min_pages=1, out=out)),
                    (5, lambda q, out: store.chunk_attention(q, cu, table, lens, 0.1, splits=splits, out=out)),
                    (200, lambda q, out: store.chunk_attention(q, 40 * cu, table, lens, 0.1, splits=splits, out=out))):
        q = _rand(gen, n, 8, 128).to(DEV)
        want = call(q, None)
        assert call(q, q) is q and torch.equal(q, want)


def test_chunk_attention_does_not_look_ahead():
    """other keys and values behind a query change nothing, bit for bit"""
    gen = _gen(2)
    n = 300
    a, table, _ = _filled(gen, [n], 2, 128)
    b = _store(a.pages.shape[0], 2, 128)
    b.pages.copy_(a.pages)
    b.exps.copy_(a.exps)
    b.pages[table[0, 10:19].long()] = 0x7E
    b.exps[table[0, 10:19].long()] = 30
    q = _rand(gen, n, 8, 128).to(DEV)
    x, y = (s.chunk_attention(q, _ints([0, n]), table, _ints([n]), 0.1) for s in (a, b))
    assert torch.equal(x[:160], y[:160]) and not torch.equal(x[160:], y[160:])


def test_chunk_of_one_token_is_a_decode_step():
    gen = _gen(8)
    lens = [100, 1, 40]
    store, table, seqs = _filled(gen, lens, 2, 128)
    q = _rand(gen, 3, 8, 128).to(DEV)
    for cu in (None, _ints([0, 1, 2, 3])):
        _check(store.chunk_attention(q, cu, table, _ints(lens), 0.1), q, seqs, [0, 1, 2, 3], lens, 0.1)


@pytest.mark.parametrize("size", [0.0, 1e-38, 1e-30, 1e30])
def test_attention_of_queries_of_any_size(size):
    """zero and tiny queries (all keys alike), huge ones"""
    gen = _gen(17)
    lens = [50, 33]
    store, table, seqs = _filled(gen, lens, 1, 64, size=1e-3)
    q = (torch.randn(70, 4, 64, generator=gen) * size).to(torch.bfloat16).to(DEV)
    scale = 0.1 if size < 1 else 1e-28
    _check(store.attention(q[:2], table, _ints(lens), scale), q[:2], seqs, [0, 1, 2], lens, scale)
    for cu in ([0, 3, 5], [0, 40, 70]):
        _check(store.chunk_attention(q[:cu[-1]], _ints(cu), table, _ints(lens), scale), q, seqs, cu, lens, scale)


@pytest.mark.parametrize("G", [33, 64])
def test_decode_attention_of_many_heads_to_one(G):
    gen = _gen(G)
    lens = [300, 1, 0, 77]
    store, table, seqs = _filled(gen, lens, 1, 128)
    q = _rand(gen, 4, G, 128, size=1.5).to(DEV)
    got = store.attention(q, table, _ints(lens), 0.09)
    assert not got[2].any()
    _check(got, q, seqs, [0, 1, 2, 3, 4], lens, 0.09)


def test_pages_beyond_four_gigabytes():
    """offsets of pages and their rows that 32 bits do not hold"""
    H, D, n = 8, 128, 40
    blocks = (1 << 32) // (H * 2 * PAGE * D) + 20
    gen = _gen(21)
    store = _store(blocks, H, D)
    last = torch.tensor([blocks - 1, 3, blocks - 7])
    p = torch.arange(n)
    K, V = _keys(gen, n, H, D), _rand(gen, n, H, D)
    for a, b in ((0, 20), (20, n)):
        store.append(K[a:b].to(DEV), V[a:b].to(DEV), (last[p[a:b] // PAGE] * PAGE + p[a:b] % PAGE).to(DEV))
    many = torch.cat([last[:1].repeat(600) * PAGE, last[p // PAGE] * PAGE + p % PAGE])       # (a long call; the last of each slot counts)
    store.append(torch.cat([K[:1].repeat(600, 1, 1), K]).to(DEV), torch.cat([V[:1].repeat(600, 1, 1), V]).to(DEV), many.to(DEV))
    assert int(store.marks.abs().max()) == 0
    ref = R.Pages(3, H, D)
    ref.append(K.double(), V.double(), p)
    kd, vd = store.dense(last.to(DEV))
    assert torch.equal(kd.cpu().double(), ref.dense()[0]) and torch.equal(vd.cpu().double(), ref.dense()[1])
    seqs = [tuple(t.flatten(0, 1)[:n] for t in ref.dense())]
    table = last[None].to(torch.int32).to(DEV)
    q = _rand(gen, 40, 16, D).to(DEV)
    _check(store.attention(q[:1], table, _ints([n]), 0.1, splits=2, min_pages=1), q[:1], seqs, [0, 1], [n], 0.1)
    for m in (3, 40):
        _check(store.chunk_attention(q[:m], _ints([0, m]), table, _ints([n]), 0.1), q[:m], seqs, [0, m], [n], 0.1)


def test_native_and_general_calls_agree(monkeypatch):
    """the same bits without the native host path"""
    gen = _gen(23)
    lens = [90, 20]
    store, table, _ = _filled(gen, lens, 2, 128)
    cos, sin = (t.to(DEV) for t in _tables(128, 100))
    K, V, q = _keys(gen, 3, 2, 128).to(DEV), _rand(gen, 3, 2, 128).to(DEV), _rand(gen, 3, 8, 128).to(DEV)
    slots = torch.tensor([int(table[0, 5]) * PAGE + 10, int(table[1, 1]) * PAGE + 4, -1], device=DEV)
    before = store.pages.clone(), store.exps.clone()

    def calls():
        store.pages.copy_(before[0])
        store.exps.copy_(before[1])
        r = store.append(K, V, slots, positions=torch.tensor([90, 20, 5], device=DEV), cos=cos, sin=sin, q=q)
        return [r, store.pages.clone(), store.exps.clone(), store.attention(r[:2], table, _ints([91, 21]), 0.1),
                store.attention(r[:2], table, _ints([91, 21]), 0.1, splits=3, window=7, starts=_ints([1, 2]), out=torch.zeros_like(r[:2])),
                store.chunk_attention(r, _ints([0, 2, 3]), table, _ints([91, 21]), 0.1), *store.dense(table[0, :3].contiguous()), *store.dense()]

    from statetree_b200 import kvcache
    assert kvcache.calls() is not None
    native = calls()
    monkeypatch.setattr(kvcache, "calls", lambda: None)
    assert all(torch.equal(a, b) for a, b in zip(native, calls()))


def test_attention_strided():
    """queries inside fused rows, an output inside a larger one, a block table that is part of a wider one"""
    gen = _gen(6)
    lens = [90, 20]
    store, table, seqs = _filled(gen, lens, 2, 128)
    big = torch.zeros(2, table.shape[1] + 5, dtype=torch.int32, device=DEV)
    big[:, 2:2 + table.shape[1]] = table
    wide = _rand(gen, 2, 12, 128).to(DEV)
    out = torch.zeros(2, 9, 128, dtype=torch.bfloat16, device=DEV)
    store.attention(wide[:, 2:10], big[:, 2:2 + table.shape[1]], _ints(lens), 0.1, out=out[:, :8])
    _check(out[:, :8], wide[:, 2:10], seqs, [0, 1, 2], lens, 0.1)
    assert not out[:, 8].any()
    out.zero_()
    store.chunk_attention(wide[:, 2:10], _ints([0, 1, 2]), big[:, 2:2 + table.shape[1]], _ints(lens), 0.1, out=out[:, :8])
    _check(out[:, :8], wide[:, 2:10], seqs, [0, 1, 2], lens, 0.1)
    assert not out[:, 8].any()


# ------------------------------------------------------------------------------------------------ streams and graphs
def test_steps_in_graphs_and_on_streams():
    """append and both attentions captured into two graphs over two stores' worth of sequences, replayed on two streams at once, equal
    the same calls made eagerly"""
    gen = _gen(12)
    H, D, n = 2, 128, 200
    results, graphs, inputs = [], [], []
    for k in range(2):
        store, table, _ = _filled(gen, [n, n - 30], H, D)
        lens = _ints([n + 1, n - 29])
        K, V, q = (_rand(gen, 2, h, D).to(DEV) for h in (H, H, 8))
        qs = _rand(gen, 24, 8, D).to(DEV)
        slots = torch.tensor([int(table[0, n // PAGE]) * PAGE + n % PAGE, int(table[1, (n - 30) // PAGE]) * PAGE + (n - 30) % PAGE], device=DEV)
        pos, (cos, sin) = torch.tensor([n, n - 30], device=DEV), (t.to(DEV) for t in _tables(D, 300))
        cu = _ints([0, 20, 24])

        def step(s=store, K=K, V=V, slots=slots, pos=pos, cos=cos, sin=sin, q=q, qs=qs, table=table, lens=lens, cu=cu):
            r = s.append(K, V, slots, positions=pos, cos=cos, sin=sin, q=q)
            return s.attention(r, table, lens, 0.1, splits=3, min_pages=1), s.chunk_attention(qs, cu, table, lens, 0.1, splits=2)

        inputs.append((store, step))
    for store, step in inputs:
        before = store.pages.clone(), store.exps.clone()
        results.append([t.clone() for t in step()])
        store.pages.copy_(before[0])
        store.exps.copy_(before[1])
    torch.cuda.synchronize()
    for store, step in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs))
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for (g, outs), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                for o in outs:
                    o.zero_()
                g.replay()
    torch.cuda.synchronize()
    for (g, outs), want in zip(graphs, results):
        assert all(torch.equal(a, b) for a, b in zip(outs, want))
    # eagerly, from both streams, on one store
    store, step = inputs[0]
    got = []
    for _ in range(4):
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                args = step.__defaults__
                got.append((store.attention(args[7], args[9], args[10], 0.1, splits=4, min_pages=1), store.chunk_attention(args[8], args[11], args[9], args[10], 0.1, splits=3)))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, got[0]))
    from statetree_b200.ops import device_status
    assert device_status() == 0
