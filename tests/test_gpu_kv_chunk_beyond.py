"""Chunk attention over lossless pages whose values hold infinities and NaN at positions that the sequences have: a query that sees them gets them, a
query that does not (a later token, one that has left its window, padding) is as it would be without them, wherever the kernel's tiles end."""
import math

import pytest
import torch

from test_gpu_kv_chunk import D, PAGE, Setup

pytestmark = pytest.mark.gpu
INF, NAN = math.inf, math.nan


def compare(s, starts=None, window=0, splits=(None, 1, 3)):
    """s's store as it is against the same store with zeros in these places: every bit, but where such a value is seen.  There: the sum of
    those seen (an infinity, NaN of NaN or of both infinities)"""
    from statetree_b200.kvcache import PageStore
    clean = PageStore(s.table.numel(), s.kv, "cuda", pool_blocks=1 << 15)
    odd = []
    for b, n in enumerate(s.lens):
        pages = s.table[b, :-(-n // PAGE)]
        K, V = (x.reshape(-1, s.kv, D)[:n].clone() for x in s.store.dense(pages))
        odd.append(torch.where(V.isfinite(), torch.zeros_like(V), V).double())
        i = torch.arange(n, device="cuda")
        clean.append(K, torch.where(V.isfinite(), V, torch.zeros_like(V)), s.table[b].long()[i // PAGE] * PAGE + i % PAGE)
    s.store.check()
    clean.check()
    dirty, G, hit = s.store, s.heads // s.kv, 0
    for sp in splits:
        got = s.call(starts=starts, window=window, splits=sp)
        s.store = clean
        want = s.call(starts=starts, window=window, splits=sp).double()
        s.store = dirty
        assert bool(want.isfinite().all())
        for b, (n, m) in enumerate(zip(s.new, s.lens)):
            at = torch.arange(m - n, m, device="cuda")[:, None]
            j = torch.arange(m, device="cuda")[None]
            seen = (j <= at) & (j >= (starts[b] if starts else 0)) & ((j > at - window) if window else (j >= 0))
            keys = (odd[b] != 0).flatten(1).any(1).nonzero()[:, 0]
            x = odd[b][keys].permute(1, 2, 0)[:, :, None]                                    # [kv, D, 1, keys]
            x = torch.where(seen[:, keys][None, None], x, 0.0).sum(-1).permute(2, 0, 1)      # [n, kv, D]
            rows = slice(int(s.cu[b]), int(s.cu[b + 1]))
            want[rows] += x.repeat_interleave(G, 1)
            hit += int((x != 0).sum())
        assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.double().nan_to_num(0, 1e300, -1e300), want.nan_to_num(0, 1e300, -1e300))
    return hit


def put(s, b, where, values):
    """values {(head, dim): value} at position `where` of sequence b"""
    V = s.V[b]
    for (h, d), x in values.items():
        V[where, h, d] = x
    first = where // PAGE * PAGE
    i = torch.arange(first, min(first + PAGE, s.lens[b]), device="cuda")
    s.store.append(s.K[b][i], V[i], s.table[b].long()[i // PAGE] * PAGE + i % PAGE)           # (the page starts over)


@pytest.mark.parametrize("new", [1, 4, 130, 300])
@pytest.mark.parametrize("value", [INF, -INF, NAN])
def test_one_value(value, new):
    """at every distance from the queries: far behind, in the tiles of 128 that the first and last of them share with it, the last key"""
    for where in sorted({0, 127, 128, 399 - new, 400 - new, 401 - new, 399}):
        if where < 400:
            s = Setup(8, 2, [new], [400], seed=where)
            put(s, 0, where, {(1, 77): value})
            assert compare(s, splits=(1, 2)) > 0


@pytest.mark.parametrize("new,lens", [([4, 3], [300, 33]), ([200, 90], [420, 300])])
@pytest.mark.parametrize("window,starts", [(0, None), (0, [70, 20]), (40, None), (1, None), (129, [250, 31])])
def test_windows_and_padding(new, lens, window, starts):
    s = Setup(12, 4, new, lens, seed=3, zeros=True)
    for b, n in enumerate(lens):
        for k, where in enumerate((0, 15, 16, 17, n // 2, n - 40, n - 3, n - 2, n - 1)):
            if 0 <= where < n:
                put(s, b, where, {(k % 4, 9 * k): INF, (k % 4, 9 * k + 1): -INF, ((k + 1) % 4, 127 - k): NAN, (3, 64 + k): [INF, -INF][k % 2]})
    assert compare(s, starts, window) > 0


def test_a_whole_row_and_both_signs():
    """rows of nothing else; an infinity of either sign in one place of two keys is NaN for who sees both"""
    for new in (6, 140):
        s = Setup(16, 2, [new], [500], seed=4)
        put(s, 0, 499, {(h, d): INF for h in range(2) for d in range(D)})
        put(s, 0, 497, {(0, d): [INF, -INF, NAN][d % 3] for d in range(D)})
        put(s, 0, 497 - new // 2, {(1, d): -INF for d in range(0, D, 5)})
        put(s, 0, 3, {(0, 0): -INF, (1, 1): INF})
        assert compare(s) > 0


def test_every_value():
    s = Setup(8, 1, [150], [150], seed=5)
    s.V[0][:] = NAN
    i = torch.arange(150, device="cuda")
    s.store.append(s.K[0], s.V[0], s.table[0].long()[i // PAGE] * PAGE + i % PAGE)
    assert compare(s, window=7) > 0


@pytest.mark.parametrize("new", [5, 260])
def test_channels(new):
    """a dimension that is an infinity or NaN in every key, others in some: all of them are found, however early the first is"""
    s = Setup(8, 2, [new], [600], seed=8)
    s.V[0][:, 0, 33], s.V[0][:, 1, 64], s.V[0][::7, 1, 127], s.V[0][300:, 0, 34] = INF, NAN, -INF, -INF
    s.V[0][595, 0, 0] = s.V[0][2, 0, 31] = NAN
    i = torch.arange(600, device="cuda")
    s.store.append(s.K[0], s.V[0], s.table[0].long()[i // PAGE] * PAGE + i % PAGE)
    assert compare(s) > 0
    assert compare(s, window=100, splits=(1, 2)) > 0


@pytest.mark.parametrize("new", [3, 70])
def test_rows_appended_again(new):
    """in place, behind entries of the row that stood there: what the pages hold is what counts"""
    s = Setup(8, 2, [new], [90], seed=6, zeros=True)
    for where in (88, 70, 33):
        s.V[0][where, 1, ::3] = torch.tensor([INF, -INF, NAN], device="cuda").repeat(15)[:43].to(torch.bfloat16)
        s.V[0][where, 0, 60:70] = -INF
        s.store.append(s.K[0][where:where + 1], s.V[0][where:where + 1], s.table[0].long()[where // PAGE:where // PAGE + 1] * PAGE + where % PAGE)
    assert compare(s) > 0


def test_a_late_chunk_in_unequal_parts():
    """a last wave that is split by itself (some units whole), values far apart over the sequence"""
    s = Setup(32, 8, [2048], [24000], seed=7, extra=0)
    for where in (1, 700, 15003, 22000, 23100, 23999):
        put(s, 0, where, {(where % 8, where % 128): NAN, (3, 5): INF})
    from statetree_b200.kvcache import chunk_splits
    assert chunk_splits(2048, 1, 8, 4, s.width)[1] > 0
    assert compare(s, splits=(None,)) > 0
