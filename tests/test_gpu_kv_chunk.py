"""PageStore.chunk_attention (causal attention of several query tokens per sequence over the lossless pages) against attention in 64 bits
over the values that were appended."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
D, PAGE = 128, 16


def kv_values(n, H, seed, dead=True, zeros=False):
    """keys with channels of different sizes (one nearly dead: an escape in every row, more than a record's eleven slots), values"""
    g = torch.Generator("cuda").manual_seed(seed)
    size = torch.randn(H, D, device="cuda", generator=g).exp()
    if dead:
        size[0, 5] = 1e-6
    K = torch.randn(n, H, D, device="cuda", generator=g) * size
    V = torch.randn(n, H, D, device="cuda", generator=g)
    if zeros:                                       # (zeros escape: chains of several blocks)
        K[:, -1, 70:110] = 0
        V[:, -1, ::3] = 0
    return K.to(torch.bfloat16), V.to(torch.bfloat16)


class Setup:
    """sequences of `lens` tokens in a store whose pages lie anywhere; q rows for the last new[b] tokens of each"""

    def __init__(self, heads, kv, new, lens, seed=0, extra=2, zeros=False, tail=0, width=None):
        from statetree_b200.kvcache import PageStore
        self.heads, self.kv, self.new, self.lens = heads, kv, new, lens
        B = len(lens)
        self.width = width or max(1, -(-max(lens) // PAGE)) + extra
        g = torch.Generator("cuda").manual_seed(seed + 99)
        blocks = B * self.width
        self.store = PageStore(blocks, kv, "cuda", pool_blocks=1 << 15)
        self.table = torch.randperm(blocks, device="cuda", generator=g).to(torch.int32).view(B, self.width)
        self.K, self.V = zip(*[kv_values(n, kv, seed + b, zeros=zeros) for b, n in enumerate(lens)]) if B else ((), ())
        for b, n in enumerate(lens):
            if n:
                i = torch.arange(n, device="cuda")
                self.store.append(self.K[b], self.V[b], self.table[b].long()[i // PAGE] * PAGE + i % PAGE)
        self.store.check()
        self.cu = torch.tensor([sum(new[:b]) for b in range(B + 1)], dtype=torch.int32, device="cuda")
        self.q = (torch.randn(sum(new) + tail, heads, D, device="cuda", generator=g) * 1.5).to(torch.bfloat16)
        self.l32 = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.scale = D ** -0.5

    def call(self, starts=None, window=0, **kw):
        s = None if starts is None else torch.tensor(starts, dtype=torch.int32, device="cuda")
        return self.store.chunk_attention(self.q, self.cu, self.table, self.l32, self.scale, starts=s, window=window, **kw)

    def check(self, out, starts=None, window=0):
        """|error| <= half a step of the output, and of P (BF16, 2^-8 of each probability), and what fp32 leaves of the scores: 128 products
        summed, 2^-22 of their magnitudes each (matrix units cut off rather than round), enters a probability and the sum that divides it"""
        for b, (n, m) in enumerate(zip(self.new, self.lens)):
            if not n:
                continue
            at = torch.arange(m - n, m, device="cuda")[:, None]
            j = torch.arange(m, device="cuda")[None]
            seen = (j <= at) & (j >= (starts[b] if starts else 0))
            if window:
                seen &= j > at - window
            rows = slice(int(self.cu[b]), int(self.cu[b + 1]))
            for h in range(self.kv):
                k, v = self.K[b][:, h].double(), self.V[b][:, h].double()
                for i in range(h * (self.heads // self.kv), (h + 1) * (self.heads // self.kv)):
                    q = self.q[rows, i].double()
                    s = (q @ k.t() * self.scale).masked_fill(~seen, -math.inf)
                    top = s.amax(1, keepdim=True)
                    p = (s - top.clamp_min(-1e300)).exp() if m else s
                    total = p.sum(1, keepdim=True)
                    p = torch.where(total > 0, p / total.clamp_min(1e-300), 0.0)
                    want, mass = p @ v, p @ v.abs()
                    size = ((q.abs() @ k.abs().t()) * self.scale * seen).amax(1, keepdim=True) if m else torch.zeros(n, 1, device="cuda").double()
                    d = 2 * 128 * 2.0 ** -22 * size + 2.0 ** -12
                    tol = 2.0 ** -8 * want.abs() + (2.0 ** -8 + d) * mass
                    off = (out[rows, i].double() - want).abs()
                    assert bool((off <= tol).all()), (b, i, float((off / tol.clamp_min(1e-30)).max()))


SHAPES = [(32, 8), (8, 8), (7, 1), (12, 4), (40, 8), (64, 1), (300, 2)]


@pytest.mark.parametrize("heads,kv", SHAPES)
@pytest.mark.parametrize("new,lens", [([1], [1]), ([5], [5]), ([3, 1, 2], [40, 1, 17]), ([1, 1], [100, 16]), ([100], [100]), ([129, 64], [400, 64]),
                                      ([257], [700]), ([0, 70, 0, 33], [20, 70, 0, 290])])
def test_chunks(heads, kv, new, lens):
    s = Setup(heads, kv, new, lens)
    for splits in (None, 1, 3):
        s.check(s.call(splits=splits))


@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 100, 127, 128, 129, 1000, (1 << 31) - 1])
@pytest.mark.parametrize("new,lens", [([4, 2], [200, 33]), ([150, 40], [420, 41])])
def test_windows(window, new, lens):
    s = Setup(8, 2, new, lens, seed=1)
    s.check(s.call(window=window), window=window)
    starts = [37, 5]
    s.check(s.call(window=window, starts=starts, splits=2), starts, window)


@pytest.mark.parametrize("new,lens,starts", [([4, 4, 4], [90, 90, 90], [0, 89, 90]), ([90, 90, 90], [90, 90, 90], [0, 17, 90]),
                                             ([200, 140], [300, 140], [128, 139]), ([2, 2], [33, 33], [32, 1000])])
def test_left_padding(new, lens, starts):
    """queries before a sequence's first token see nothing: zeros"""
    s = Setup(16, 4, new, lens, seed=2)
    for splits in (1, 4):
        out = s.call(starts=starts, splits=splits)
        s.check(out, starts)
        for b, first in enumerate(starts):
            pos = torch.arange(lens[b] - new[b], lens[b], device="cuda")
            assert bool((out[int(s.cu[b]):int(s.cu[b + 1])][pos < first] == 0).all())


@pytest.mark.parametrize("new", [3, 90])
def test_sequences_shorter_than_their_queries(new):
    """positions below zero see nothing; lens of zero"""
    s = Setup(8, 2, [new, new], [new, new], seed=3)
    s.l32 = torch.tensor([new - 2, 0], dtype=torch.int32, device="cuda")
    out = s.call()
    assert bool((out[:2] == 0).all()) and bool((out[new:] == 0).all())
    t = Setup(8, 2, [new - 2, 0], [new - 2, 0], seed=3)
    t.K, t.V, t.table, t.store, t.q = [s.K[0][:new - 2], s.K[1][:0]], [s.V[0][:new - 2], s.V[1][:0]], s.table, s.store, s.q[2:]
    t.check(out[2:])


@pytest.mark.parametrize("new", [6, 140])
def test_escapes_and_chains(new):
    """zeros in many channels: records whose escapes fill several blocks of the pool; values come back exactly: the one key of a sequence
    of one token returns its values"""
    s = Setup(8, 4, [new, new], [500, 300], seed=4, zeros=True)
    assert s.store.pool_usage()[0] > 100
    s.check(s.call())
    flat = Setup(8, 4, [1], [1], seed=4, zeros=True)
    out = flat.call()                                                     # one key: P is 1
    assert torch.equal(out[0].view(4, 2, D)[:, 0], flat.V[0][0]) and torch.equal(out[0].view(4, 2, D)[:, 1], flat.V[0][0])


@pytest.mark.parametrize("heads,kv,new,lens", [(8, 2, [300, 7, 0, 200], [400, 300, 9, 260]), (4, 2, [5, 3], [200, 90])])
@pytest.mark.parametrize("whole", [1, 2, 5, 1000])
def test_units_that_are_not_split(heads, kv, new, lens, whole, monkeypatch):
    """some units whole, the others split, ragged; both host paths; rows behind the last sequence"""
    from statetree_b200 import kvcache
    s = Setup(heads, kv, new, lens, seed=16, tail=3)
    for splits in (2, 3):
        monkeypatch.setattr(kvcache, "chunk_splits", lambda *a: (splits, whole))
        buf = torch.full((s.q.shape[0], heads, D), 3.0, dtype=torch.bfloat16, device="cuda")
        s.check(s.call(out=buf))
        assert bool((buf[sum(new):] == 3).all())
        native = kvcache.calls
        monkeypatch.setattr(kvcache, "calls", lambda: None)
        assert torch.equal(s.call()[:sum(new)], buf[:sum(new)])
        monkeypatch.setattr(kvcache, "calls", native)


@pytest.mark.parametrize("new", [4, 90])
@pytest.mark.parametrize("tiny", [3, 14, 40])
def test_rows_that_were_appended_again(new, tiny):
    """a row rewritten in place leaves its old escapes in the list, before the new ones of the same elements: the attention reads what the
    pages decode to (tiny escapes a row and half: in the unit's slots, beyond them, and in chains)"""
    s = Setup(8, 2, [new], [200], seed=14)
    i = torch.arange(200, device="cuda")
    slots = s.table[0].long()[i // PAGE] * PAGE + i % PAGE
    K, V = kv_values(200, 2, 5, dead=False)
    for t in (K, V):
        t[:, :, :tiny] = (t[:, :, :tiny].float() * 1e-7).to(torch.bfloat16)
    s.store.append(K, V, slots)
    again = torch.tensor([17, 18, 37, 190, 199], device="cuda")             # (not the first of their pages)
    for times in range(2):
        for t in (K, V):
            t[again] = (t[again].float() * -1.5).to(torch.bfloat16)
        for j in again.tolist():
            s.store.append(K[j:j + 1], V[j:j + 1], slots[j:j + 1])
    s.store.check()
    Kd, Vd = s.store.dense()
    Kd, Vd = Kd.view(-1, 2, D)[slots], Vd.view(-1, 2, D)[slots]
    assert torch.equal(Kd, K) and torch.equal(Vd, V)
    s.K, s.V = [Kd], [Vd]
    for splits in (1, 3):
        s.check(s.call(splits=splits))
    one = Setup(8, 2, [1], [1], seed=15)                                    # one key: its value comes back exactly
    one.store, one.table, one.l32 = s.store, (slots[199:200] // PAGE).int()[None], torch.tensor([16], dtype=torch.int32, device="cuda")
    start = torch.tensor([int(slots[199] % PAGE)], dtype=torch.int32, device="cuda")
    one.l32 = start + 1
    out = one.store.chunk_attention(one.q, one.cu, one.table, one.l32, one.scale, starts=start)
    assert torch.equal(out[0].view(2, 4, D), V[199][:, None].expand(2, 4, D))


@pytest.mark.parametrize("new", [3, 70])
@pytest.mark.parametrize("junk", [float("nan"), float("inf"), -float("inf"), 3e38])
def test_values_in_masked_places(new, junk):
    """rows of the pages before starts and behind lens may hold anything: NaN, infinities, the type's largest"""
    s = Setup(8, 2, [new, new], [170, 150], seed=5)
    from statetree_b200.kvcache import PageStore
    store = PageStore(s.table.numel(), 2, "cuda", pool_blocks=1 << 15)
    starts, keep = [40, 21], [160, 133]
    for b, n in enumerate(s.lens):
        K, V = s.K[b].clone(), s.V[b].clone()
        for t in (K, V):
            t[:starts[b]] = junk
            t[keep[b]:] = junk
        i = torch.arange(n, device="cuda")
        store.append(K, V, s.table[b].long()[i // PAGE] * PAGE + i % PAGE)
    s.store, s.lens = store, keep
    s.K, s.V = [k[:n] for k, n in zip(s.K, keep)], [v[:n] for v, n in zip(s.V, keep)]
    s.l32 = torch.tensor(keep, dtype=torch.int32, device="cuda")
    for splits in (1, 2):
        out = s.call(starts=starts, splits=splits)
        assert bool(torch.isfinite(out).all())
        s.check(out, starts)


@pytest.mark.parametrize("new", [2, 80])
def test_a_query_that_is_no_number(new):
    """its row alone is none"""
    s = Setup(8, 2, [new], [300], seed=6)
    clean = s.call()
    s.q[1, 3, 7] = float("nan")
    out = s.call()
    assert bool(torch.isnan(out[1, 3]).all())
    out[1, 3] = clean[1, 3]
    assert torch.equal(out, clean)


@pytest.mark.parametrize("new", [2, 90])
def test_block_tables(new):
    """part of a wider table, one row for all sequences, entries that are no pages where nothing is read, keys beyond the table"""
    s = Setup(8, 2, [new, new], [250, 250], seed=7)
    want = s.call()
    wide = torch.full((2, 40), -7, dtype=torch.int32, device="cuda")
    wide[:, 3:3 + s.width] = s.table
    table, s.table = s.table, wide[:, 3:3 + s.width]
    assert not s.table.is_contiguous() and torch.equal(s.call(), want)
    s.table = table.clone()
    s.table[:, 250 // PAGE + 1:] = 1 << 30                                 # (behind the last key)
    assert torch.equal(s.call(), want)
    s.table = table[:1].expand(2, -1)
    one = s.call()
    assert torch.equal(one[:new], want[:new])
    s.K, s.V = (s.K[0], s.K[0]), (s.V[0], s.V[0])
    s.check(one)
    # a table that ends before the sequence does: what is beyond it takes no part
    s.table = table[:, :10].contiguous()
    short = s.call(splits=1)
    t = Setup(8, 2, [new], [160], seed=7)
    k = s.K[0][:160].double()
    for i in (0, new - 1):                                                  # (all of these positions are behind the table)
        if 250 - new + i < 160:
            continue
        for h in range(8):
            p = torch.softmax(s.q[i, h].double() @ k[:, h // 4].t() * s.scale, 0)
            v = s.V[0][:160, h // 4].double()
            assert bool(((short[i, h].double() - p @ v).abs() <= 2.0 ** -8 * (p @ v).abs() + 2.0 ** -7 * (p @ v.abs())).all())
    assert t.width > 0


@pytest.mark.parametrize("new", [4, 100])
def test_given_outputs_and_rows_behind(new):
    """out as part of a wider buffer; rows behind the last sequence stay as they were; q at a token stride, heads contiguous"""
    s = Setup(8, 2, [new, new], [300, 270], seed=8, tail=5)
    buf = torch.full((2 * new + 5, 11, D), 7.0, dtype=torch.bfloat16, device="cuda")
    for splits in (1, 3):
        buf.fill_(7.0)
        out = s.call(out=buf[:, 2:10], splits=splits)
        s.check(out)
        assert bool((buf[2 * new:] == 7).all()) and bool((buf[:, :2] == 7).all()) and bool((buf[:, 10:] == 7).all())
    qkv = torch.randn(2 * new + 5, 12, D, device="cuda").to(torch.bfloat16)
    qkv[:, :8] = s.q
    s.q = qkv[:, :8]
    s.check(s.call())
    odd = torch.zeros(2 * new + 5, 8 * D + 1, dtype=torch.bfloat16, device="cuda")       # (copied: its rows are not 16-byte aligned)
    odd[:, 1:] = s.q.flatten(1)
    s.q = odd[:, 1:].unflatten(1, (8, D))
    s.check(s.call())


def test_one_query_each_agrees_with_the_decode_attention():
    s = Setup(32, 8, [1] * 9, [1, 15, 16, 17, 33, 200, 640, 900, 31], seed=9)
    a = s.store.chunk_attention(s.q, None, s.table, s.l32, s.scale)
    s.check(a)
    b = s.store.attention(s.q, s.table, s.l32, s.scale)
    s.check(b)


@pytest.mark.parametrize("new", [3, 130])
def test_graph_and_streams(new):
    """captured once, replayed after more tokens have come in and queries have changed; a call on another stream meanwhile"""
    s = Setup(16, 4, [new, new], [400, 390], seed=10)
    side, lens = torch.cuda.Stream(), list(s.lens)
    side.wait_stream(torch.cuda.current_stream())
    s.l32.fill_(200)
    with torch.cuda.stream(side):
        s.call(splits=3)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = s.call(splits=3)
    torch.cuda.current_stream().wait_stream(side)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    for now in ([400, 390], [new, 250]):
        s.l32.copy_(torch.tensor(now, dtype=torch.int32, device="cuda"))
        s.q.normal_()
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            side_out = s.call(splits=3)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, side_out)
        K, V = s.K, s.V
        s.K, s.V, s.lens = [k[:n] for k, n in zip(K, now)], [v[:n] for v, n in zip(V, now)], now
        s.check(out)
        s.K, s.V, s.lens = K, V, lens


def test_the_same_call_twice_gives_the_same_bits():
    s = Setup(32, 8, [70, 3, 300], [900, 500, 300], seed=11)
    a = s.call()
    for _ in range(5):
        assert torch.equal(s.call(), a)


def test_far_pages():
    """a page beyond 2^32 bytes of the cache"""
    from statetree_b200.kvcache import PageStore
    blocks = (1 << 32) // 6400 + 64
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GB")
    store = PageStore(blocks, 1, "cuda")
    for new in (3, 140):
        n = 150
        K, V = kv_values(n, 1, new)
        pages = torch.arange(blocks - 10, blocks, device="cuda")
        i = torch.arange(n, device="cuda")
        store.append(K, V, pages[i // PAGE] * PAGE + i % PAGE)
        s = Setup.__new__(Setup)
        s.heads, s.kv, s.new, s.lens, s.K, s.V, s.store = 4, 1, [new], [n], [K], [V], store
        s.table, s.cu = pages.int()[None], torch.tensor([0, new], dtype=torch.int32, device="cuda")
        s.q, s.l32, s.scale = torch.randn(new, 4, D, device="cuda").to(torch.bfloat16), torch.tensor([n], dtype=torch.int32, device="cuda"), D ** -0.5
        s.check(s.call())


def test_empty_calls_and_refusals():
    s = Setup(8, 2, [3, 3], [20, 30], seed=12)
    st, q, cu, tb, ln = s.store, s.q, s.cu, s.table, s.l32
    assert st.chunk_attention(q[:0], cu * 0, tb, ln, 1.0).shape == (0, 8, D)
    bad = [dict(q=q.float()), dict(q=q[:, :7]), dict(q=q[..., :64]), dict(cu=cu.long()), dict(cu=cu[:2]), dict(table=tb.long()), dict(table=tb[0]),
           dict(lens=ln.long()), dict(lens=ln[:1]), dict(scale=0.0), dict(scale=-1.0), dict(scale=600.0), dict(splits=0), dict(splits=2000),
           dict(window=-1), dict(starts=ln.long()), dict(starts=ln[:1]), dict(out=q.float()), dict(out=torch.empty_like(q)[:5]),
           dict(out=torch.empty_like(q)[:1].expand(6, 8, D)), dict(q=q.cpu()), dict(lens=ln.cpu()), dict(cu=None)]
    for kw in bad:
        a = dict(q=q, cu=cu, table=tb, lens=ln, scale=s.scale, splits=None, starts=None, out=None, window=0)
        a.update(kw)
        with pytest.raises((RuntimeError, IndexError)):
            st.chunk_attention(a["q"], a["cu"], a["table"], a["lens"], a["scale"], splits=a["splits"], starts=a["starts"], out=a["out"],
                               window=a["window"])
    s.check(s.call())


def test_store_over_tensors():
    from statetree_b200.kvcache import PageStore
    s = Setup(8, 2, [3], [50], seed=13, zeros=True)
    over = PageStore.over(s.store.pages, s.store.pool)
    assert torch.equal(over.chunk_attention(s.q, s.cu, s.table, s.l32, s.scale), s.call())
    for a, b in zip(over.dense(), s.store.dense()):
        assert torch.equal(a, b)
    with pytest.raises(RuntimeError):
        PageStore.over(s.store.pages[..., :1599], s.store.pool)
    with pytest.raises(RuntimeError):
        PageStore.over(s.store.pages, s.store.pool.long())
