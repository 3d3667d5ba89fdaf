"""The 8-bit paged KV cache as measurable cases: keys and values appended to its pages with the position rotation on the way,
and attention that reads those pages, for one query token per sequence and for ragged chunks of them.

A page holds 16 tokens of one layer: codes uint8 [blocks, KV heads, 2 (keys, values), 16, dim], each an e4m3 number, and
exps int8 [blocks, KV heads, 2]; a code stands for e4m3(code) * 2^exp.  exp is the smallest integer in [-64, 56] under which the
block's largest value is at most 448.  At dim 128 the 16-byte pieces of a row lie in another order: piece c of row r at place
c ^ (r & 6) ^ 4 (r & 1).

`kind` names the path:

  append  new tokens of `seqs` sequences (fused q/k/v rows as a projection leaves them): per-head RMSNorm (`norm`), rotation of
          queries and keys by the tokens' positions, keys and values into the pages (whose last page is partly filled), and the
          pages read back as dense BF16
  decode  attention of one new token per sequence
  chunk   causal attention of up to `new` tokens per sequence that stand at the end of up to `ctx` cached ones

Lengths depend on the case alone (`ragged`: spread over the range, some sequences of a chunk without tokens), values on the seed.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
PAGE = 16
E_MIN, E_MAX = -64, 56


def listed():
    return [
        # a decode step of one user: the smallest call, latency counts
        dict(name="append_step_b1", kind="append", seqs=1, new=1, ragged=False, heads=32, kv_heads=8, dim=128, pairs=True, norm=True),
        # a decode step of many users
        dict(name="append_step_b192", kind="append", seqs=192, new=1, ragged=False, heads=28, kv_heads=4, dim=128, pairs=False, norm=False),
        # prompt chunks of several users whose last pages are partly filled, small heads
        dict(name="append_ragged_d64", kind="append", seqs=7, new=333, ragged=True, heads=14, kv_heads=2, dim=64, pairs=False, norm=False),
        # long prompts
        dict(name="append_prompt_32k", kind="append", seqs=4, new=8191, ragged=False, heads=32, kv_heads=8, dim=128, pairs=True, norm=True),
        # one user with a short conversation
        dict(name="decode_b1_1k", kind="decode", seqs=1, ctx=1000, ragged=False, heads=32, kv_heads=8, dim=128, window=0, pad=0),
        # one user with a very long one: the work has to be split over the cache
        dict(name="decode_b1_60k", kind="decode", seqs=1, ctx=61003, ragged=False, heads=32, kv_heads=8, dim=128, window=0, pad=0),
        # many users, contexts of different lengths
        dict(name="decode_b64_8k", kind="decode", seqs=64, ctx=8192, ragged=True, heads=32, kv_heads=8, dim=128, window=0, pad=0),
        # a sliding window and left-padded sequences, small heads, seven query heads per KV head
        dict(name="decode_b33_window_d64", kind="decode", seqs=33, ctx=5000, ragged=True, heads=14, kv_heads=2, dim=64, window=1024, pad=77),
        # speculative tokens of a few users
        dict(name="chunk_b8_t4", kind="chunk", seqs=8, new=4, ctx=2900, ragged=False, heads=32, kv_heads=8, dim=128, window=0),
        # a prompt from its beginning
        dict(name="chunk_prompt_4k", kind="chunk", seqs=1, new=4096, ctx=0, ragged=False, heads=32, kv_heads=8, dim=128, window=0),
        # chunks of different lengths over different contexts, small heads
        dict(name="chunk_ragged_d64", kind="chunk", seqs=9, new=700, ctx=2500, ragged=True, heads=14, kv_heads=2, dim=64, window=900),
        # a late chunk of a very long prompt
        dict(name="chunk_2k_over_30k", kind="chunk", seqs=1, new=2048, ctx=30000, ragged=False, heads=32, kv_heads=8, dim=128, window=0),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(("append", "decode", "chunk"))
    heads, kv, dim = rng.choice(((32, 8, 128), (28, 4, 128), (14, 2, 64), (16, 16, 128), (8, 1, 128), (40, 8, 128), (12, 1, 64),
                                 (16, 8, 64), (9, 3, 128), (64, 8, 64)))
    d = dict(kind=kind, heads=heads, kv_heads=kv, dim=dim, ragged=rng.random() < 0.6)
    if kind == "append":
        seqs = _log(rng, 1, 256)
        return dict(d, seqs=seqs, new=_log(rng, 1, max(1, 16384 // seqs)), pairs=rng.random() < 0.5, norm=rng.random() < 0.5)
    window = rng.choice((0, 0, 0, 1, 100, 777, 4096))
    if kind == "decode":
        seqs = _log(rng, 1, 128)
        return dict(d, seqs=seqs, ctx=_log(rng, 1, min(65536, 262144 * 8 // (kv * seqs))), window=window, pad=rng.choice((0, 0, 5, 200)))
    seqs = _log(rng, 1, 24)
    new = _log(rng, 1, 4096 // seqs)
    return dict(d, seqs=seqs, new=new, ctx=_log(rng, 1, min(32768, (1 << 30) // (seqs * new * heads) + 16, 262144 // seqs)), window=window)


# ------------------------------------------------------------------------------------------------ lengths, work
def _spread(c, lo, hi, salt):
    """a length per sequence: all `hi`, or spread over [lo, hi] by the golden ratio, the first one `hi`"""
    if not c["ragged"]:
        return [hi] * c["seqs"]
    return [hi if b == 0 else lo + int((b * 0.6180339887498949 + salt) % 1.0 * (hi - lo + 1)) for b in range(c["seqs"])]


def _append_lens(c):
    """(new tokens, tokens that the last page holds already, position of the first new token) per sequence"""
    new = _spread(c, 1, c["new"], 0.3)
    held = [(5 * b + 11) % PAGE for b in range(c["seqs"])]
    first = [h + 16 * ((37 * b) % 400) if c["new"] < 4096 else h for b, h in enumerate(held)]
    return new, held, first


def _decode_lens(c):
    lens = _spread(c, 0, c["ctx"], 0.7)
    return lens, [min(n, c["pad"] * (b % 2)) for b, n in enumerate(lens)]


def _chunk_lens(c):
    new, old = _spread(c, 0, c["new"], 0.1), _spread(c, 0, c["ctx"], 0.5)
    return new, [n + o for n, o in zip(new, old)]


def work(case):
    c = case
    hq, h, D = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "append":
        new, held, _ = _append_lens(c)
        n, pages = sum(new), sum(-(-(a + b) // PAGE) for a, b in zip(new, held))
        return dict(bytes=n * (hq + 2 * h) * D * 2 + n * D * 4 + n * hq * D * 2 + n * 2 * h * D + pages * h * 2 * PAGE * D * 3,
                    flops=n * (hq + h) * D * 4)
    win = c["window"] or 1 << 60
    if c["kind"] == "decode":
        lens, starts = _decode_lens(c)
        seen = [max(0, n - max(s, n - win)) for n, s in zip(lens, starts)]
        return dict(bytes=sum(seen) * h * 2 * D + 4 * c["seqs"] * hq * D, flops=4 * D * hq * sum(seen))
    new, lens = _chunk_lens(c)
    seen = cached = 0
    for n, m in zip(new, lens):
        seen += sum(min(win, p + 1) for p in range(m - n, m))
        cached += min(m, n - 1 + win) if n else 0
    return dict(bytes=cached * h * 2 * D + 4 * sum(new) * hq * D, flops=4 * D * hq * seen)


# ------------------------------------------------------------------------------------------------ inputs
def _keys(shape, gen):
    """keys: N(0, 1) times a spread of channel sizes (LogNormal(0, 1)), as projections produce them"""
    size = torch.randn(shape[-2:], device=DEV, generator=gen).exp()
    return torch.randn(shape, device=DEV, generator=gen) * size


def _exponent(top):
    """the smallest e in [E_MIN, E_MAX] with top <= 448 * 2^e"""
    m, k = torch.frexp(top)
    return torch.where(top > 0, torch.where(m > 0.875, k - 8, k - 9), torch.full_like(k, E_MIN)).clamp(E_MIN, E_MAX)


def _codes(x, e):
    return torch.ldexp(x, -e).clamp(-448, 448).to(torch.float8_e4m3fn)


def _order(t):
    """rows of 16-byte pieces [..., 16, dim] into the order that a page keeps, or back (it is its own inverse)"""
    if t.shape[-1] != 128:
        return t
    r, c = torch.arange(PAGE, device=t.device)[:, None], torch.arange(8, device=t.device)[None]
    at = c ^ (r & 6) ^ (4 * (r & 1))
    v = t.unflatten(-1, (8, 16))
    return torch.gather(v, -2, at[..., None].expand(v.shape)).flatten(-2)


def _page_set(K, V):
    """float32 K, V [pages, 16, heads, dim] as pages: (codes, exps)"""
    x = torch.stack([K, V], 1).permute(0, 3, 1, 2, 4)                            # [pages, heads, 2, 16, dim]
    e = _exponent(x.abs().amax((-1, -2)))
    return _order(_codes(x, e[..., None, None]).view(torch.uint8)).contiguous(), e.to(torch.int8)


def _store(state):
    """the handle that a user's program keeps: the framework's store over these pages"""
    if own:
        pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "statetree-representation_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from statetree_b200.kvcache import PageStore8
        state["store"] = PageStore8.over(state["pages"], state["exps"])
    return state


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(1 + int(seed))
    hq, h, D = c["heads"], c["kv_heads"], c["dim"]
    ints = lambda v, t=torch.int32: torch.tensor(v, dtype=t, device=DEV)                      # noqa: E731
    if c["kind"] == "append":
        new, held, first = _append_lens(c)
        n, per = sum(new), [-(-(a + b) // PAGE) for a, b in zip(new, held)]
        pages = sum(per)
        order = torch.randperm(pages, device=DEV, generator=gen)                             # a sequence's pages lie anywhere
        page0 = [sum(per[:b]) for b in range(c["seqs"])]
        seq = torch.repeat_interleave(torch.arange(c["seqs"], device=DEV), ints(new, torch.long))
        i = torch.arange(n, device=DEV) - ints([sum(new[:b]) for b in range(c["seqs"])], torch.long)[seq]
        at = ints(held, torch.long)[seq] + i
        slots = order[ints(page0, torch.long)[seq] + at // PAGE] * PAGE + at % PAGE
        qkv = torch.cat([torch.randn(n, hq, D, device=DEV, generator=gen), _keys((n, h, D), gen),
                         torch.randn(n, h, D, device=DEV, generator=gen)], 1).to(torch.bfloat16).flatten(1)
        old = torch.zeros(2, pages, PAGE, h, D, device=DEV)                                  # what the last pages hold already
        begin, rows = order[ints(page0, torch.long)], torch.arange(PAGE, device=DEV)
        live = rows[None] < ints(held)[:, None]
        for x, make in ((old[0], _keys), (old[1], lambda s, g: torch.randn(s, device=DEV, generator=g))):
            x[begin] = make((c["seqs"], PAGE, h, D), gen) * live[..., None, None]
        codes, exps = _page_set(old[0], old[1])
        span = max(f + a for f, a in zip(first, new))
        inv = 1e6 ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
        ang = torch.arange(span, device=DEV, dtype=torch.float64)[:, None] * inv
        w = [1 + 0.1 * torch.randn(D, device=DEV, generator=gen) for _ in range(2)]
        return _store(dict(case=c, pages=codes, exps=exps, qkv=qkv, slots=slots, positions=ints(first, torch.long)[seq] + i,
                           cos=ang.cos().float(), sin=ang.sin().float(), blocks=order.to(torch.int32),
                           wq=w[0].to(torch.bfloat16) if c["norm"] else None, wk=w[1].to(torch.bfloat16) if c["norm"] else None))
    new, lens = _chunk_lens(c) if c["kind"] == "chunk" else ([1] * c["seqs"], _decode_lens(c)[0])
    width = max(1, -(-max(lens) // PAGE))
    pages = c["seqs"] * width
    codes = torch.empty(pages, h, 2, PAGE, D, dtype=torch.uint8, device=DEV)
    exps = torch.empty(pages, h, 2, dtype=torch.int8, device=DEV)
    step = max(1, (1 << 28) // (PAGE * h * D))
    size = torch.randn(h, D, device=DEV, generator=gen).exp()
    for p in range(0, pages, step):                                                          # (a large cache is filled in parts)
        shape = (min(step, pages - p), PAGE, h, D)
        codes[p:p + step], exps[p:p + step] = _page_set(torch.randn(shape, device=DEV, generator=gen) * size,
                                                        torch.randn(shape, device=DEV, generator=gen))
    q = torch.randn(sum(new), hq, D, device=DEV, generator=gen) * 1.5
    state = dict(case=c, pages=codes, exps=exps, q=q.to(torch.bfloat16), lens=ints(lens), scale=D ** -0.5,
                 table=torch.randperm(pages, device=DEV, generator=gen).to(torch.int32).view(c["seqs"], width))
    if c["kind"] == "chunk":
        state.update(cu=ints([sum(new[:b]) for b in range(c["seqs"] + 1)]), longest=max(new))
    else:
        state["starts"] = ints(_decode_lens(c)[1]) if c["pad"] else None
    return _store(state)


# ------------------------------------------------------------------------------------------------ one pass
def _values(pages, exps):
    """pages as the float32 values that they stand for [blocks, heads, 2, 16, dim]"""
    return torch.ldexp(_order(pages).view(torch.float8_e4m3fn).float(), exps[..., None, None].int())


def _rotated(x, w, cos, sin, pairs):
    """float32 x [tokens, heads, dim]: RMSNorm with weights w (None: none), then the rotation"""
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    a, b = (x[..., 0::2], x[..., 1::2]) if pairs else x.chunk(2, -1)
    y = a * cos - b * sin, a * sin + b * cos
    return torch.stack(y, -1).flatten(-2) if pairs else torch.cat(y, -1)


def _append(s):
    c = s["case"]
    hq, h, D = c["heads"], c["kv_heads"], c["dim"]
    n = s["qkv"].shape[0]
    q, k, v = s["qkv"].view(n, hq + 2 * h, D).split([hq, h, h], 1)
    if own:
        q = s["store"].append(k, v, s["slots"], positions=s["positions"], cos=s["cos"], sin=s["sin"], interleaved=c["pairs"], q=q,
                              q_norm=s["wq"], k_norm=s["wk"], eps=1e-6)
        kd, vd = s["store"].dense(s["blocks"])
        return dict(q=q, k=kd, v=vd)
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    kv = torch.stack([_rotated(k.float(), s["wk"], cos, sin, c["pairs"]), v.float()], 2)     # [tokens, heads, 2, dim]
    page, row = s["slots"] // PAGE, s["slots"] % PAGE
    x = _values(s["pages"], s["exps"])
    written = torch.zeros(x.shape[0], PAGE, dtype=torch.bool, device=DEV)
    written[page, row] = True
    anew = written[:, 0]                                                                     # a page that is written from its first row
    x = torch.where(anew[:, None, None, None, None], torch.zeros_like(x), x)
    x[page, :, :, row] = kv
    e = _exponent((x.abs() * written[:, None, None, :, None]).amax((-1, -2)))
    e = torch.where(anew[:, None, None], e, torch.maximum(e, s["exps"].int()))[..., None, None]
    x = torch.ldexp(_codes(x, e).float(), e).to(torch.bfloat16)[s["blocks"].long()]
    return dict(q=_rotated(q.float(), s["wq"], cos, sin, c["pairs"]).to(torch.bfloat16), k=x[:, :, 0].transpose(1, 2).contiguous(),
                v=x[:, :, 1].transpose(1, 2).contiguous())


def _attend(s, q, at, starts):
    """float32 q [seqs, n, heads, dim] at positions `at` [seqs, n] (negative: no query) over the pages"""
    c = s["case"]
    B, n, hq, D = q.shape
    h, width = c["kv_heads"], s["table"].shape[1]
    x = _values(s["pages"][s["table"].long()], s["exps"][s["table"].long()])                 # [seqs, pages, heads, 2, 16, dim]
    k, v = (x[:, :, :, i].transpose(1, 2).reshape(B, h, width * PAGE, D) for i in range(2))
    del x
    S = torch.matmul(q.view(B, n, h, hq // h, D).permute(0, 2, 1, 3, 4).reshape(B, h, n * (hq // h), D) * s["scale"], k.transpose(2, 3))
    j = torch.arange(width * PAGE, device=DEV)
    seen = (j <= at[..., None]) & (j >= starts[:, None, None])
    if c["window"]:
        seen &= j > at[..., None] - c["window"]
    S = S.view(B, h, n, hq // h, -1).masked_fill_(~seen[:, None, :, None], float("-inf")).view(S.shape)
    top = S.amax(-1, keepdim=True).clamp_min(-3e38)                                          # (a row that sees nothing: sums of zero)
    P = S.sub_(top).exp_()
    o = torch.matmul(P, v) / P.sum(-1, keepdim=True).clamp_min(1e-30)
    return o.view(B, h, n, hq // h, D).permute(0, 2, 1, 3, 4).reshape(B, n, hq, D)


def run(state):
    s = state
    c = s["case"]
    if c["kind"] == "append":
        return _append(s)
    if c["kind"] == "decode":
        if own:
            return s["store"].attention(s["q"], s["table"], s["lens"], s["scale"], starts=s["starts"], window=c["window"])
        starts = s["starts"] if s["starts"] is not None else torch.zeros_like(s["lens"])
        return _attend(s, s["q"].float()[:, None], s["lens"][:, None] - 1, starts)[:, 0].to(torch.bfloat16)
    if own:
        return s["store"].chunk_attention(s["q"], s["cu"], s["table"], s["lens"], s["scale"], window=c["window"])
    new = s["cu"][1:] - s["cu"][:-1]
    i = torch.arange(s["longest"], device=DEV)
    live = i[None] < new[:, None]                                                            # rows of the padded batch that are queries
    row = (s["cu"][:-1, None] + i).clamp_max(s["q"].shape[0] - 1)
    at = torch.where(live, (s["lens"] - new)[:, None] + i, -1)
    o = _attend(s, s["q"][row.long()].float(), at, torch.zeros_like(s["lens"]))
    out = torch.empty_like(s["q"])
    seq = torch.searchsorted(s["cu"][1:], torch.arange(s["q"].shape[0], device=DEV, dtype=torch.int32), right=True)
    out.copy_(o[seq, torch.arange(s["q"].shape[0], device=DEV) - s["cu"][seq]])
    return out


# ------------------------------------------------------------------------------------------------ in 64 bits
_LEVELS = sorted({m * 2.0 ** (e - 10) if e else m * 2.0 ** -9 for e in range(16) for m in (range(8, 16) if e else range(8))} - {480.0})


def _e4m3(x):
    """float64 x to the nearest e4m3 number (ties to the even one of its two neighbours), by search in the list of them"""
    lev = torch.tensor(_LEVELS, dtype=torch.float64, device=x.device)
    a = x.abs().clamp_max(448)
    hi = torch.searchsorted(lev, a).clamp(1, len(_LEVELS) - 1)
    lo = hi - 1
    dl, dh = a - lev[lo], lev[hi] - a
    pick = torch.where((dh < dl) | ((dh == dl) & (hi % 2 == 0)), hi, lo)
    return lev[pick].copysign(x)


def _exact_append(c, s):
    hq, h, D = c["heads"], c["kv_heads"], c["dim"]
    x = s["qkv"].double().view(-1, hq + 2 * h, D)
    n = x.shape[0]
    inv = 1e6 ** (-torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
    turn = torch.polar(torch.ones(n, D // 2, dtype=torch.float64, device=DEV), s["positions"].double()[:, None] * inv)[:, None]

    def rot(y, w):
        if w is not None:
            y = y / (y.pow(2).sum(-1, keepdim=True) / D + 1e-6).sqrt() * w.double()
        z = torch.complex(y[..., 0::2].contiguous(), y[..., 1::2].contiguous()) if c["pairs"] else torch.complex(y[..., :D // 2].contiguous(), y[..., D // 2:].contiguous())
        z = z * turn
        return torch.view_as_real(z).flatten(-2) if c["pairs"] else torch.cat([z.real, z.imag], -1)

    out = [rot(x[:, :hq], s["wq"])]
    blocks = s["blocks"].long()
    anew = torch.zeros(s["pages"].shape[0], dtype=torch.bool, device=DEV)
    anew[s["slots"][s["slots"] % PAGE == 0] // PAGE] = True
    for i, y in enumerate((rot(x[:, hq:hq + h], s["wk"]), x[:, hq + h:])):
        e_old = s["exps"][:, :, i].double()
        old = _order(s["pages"][:, :, i]).view(torch.float8_e4m3fn).double() * torch.exp2(e_old)[..., None, None]
        flat = old.transpose(1, 2).reshape(-1, h, D) * (~anew).repeat_interleave(PAGE)[:, None, None]
        flat[s["slots"]] = y
        fresh = torch.zeros_like(flat)
        fresh[s["slots"]] = y
        top = fresh.view(-1, PAGE, h, D).abs().amax((1, 3))
        e = torch.ceil(torch.log2((top / 448).clamp_min(2.0 ** E_MIN))).clamp(E_MIN, E_MAX)
        e = torch.where(top > 448 * torch.exp2(e), e + 1, torch.where(top <= 448 * torch.exp2(e - 1), e - 1, e)).clamp_min(E_MIN)   # (log2 is rounded)
        e = torch.where(anew[:, None], e, torch.maximum(e, e_old))
        step = torch.exp2(e)[:, None, :, None]
        out.append((_e4m3(flat.view(-1, PAGE, h, D) / step) * step)[blocks])
    return dict(q=out[0], k=out[1], v=out[2])


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    if c["kind"] == "append":
        return _exact_append(c, s)
    decode = c["kind"] == "decode"
    hq, h, D = c["heads"], c["kv_heads"], c["dim"]
    lens, starts = s["lens"].tolist(), s["starts"].tolist() if decode and s["starts"] is not None else [0] * c["seqs"]
    cu = list(range(c["seqs"] + 1)) if decode else s["cu"].tolist()
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, (m, first) in enumerate(zip(lens, starts)):
        n = cu[b + 1] - cu[b]
        pages = s["table"][b, :-(-m // PAGE)].long()
        if n == 0 or m == 0:
            continue
        at = torch.arange(m - n, m, device=DEV)[:, None]
        j = torch.arange(m, device=DEV)[None]
        hide = (j > at) | (j < first) | ((j <= at - c["window"]) if c["window"] else j < 0)
        for g in range(h):
            kv = (_order(s["pages"][pages, g]).view(torch.float8_e4m3fn).double() * torch.exp2(s["exps"][pages, g].double())[..., None, None])
            k, v = kv[:, 0].reshape(-1, D)[:m], kv[:, 1].reshape(-1, D)[:m]
            for i in range(g * (hq // h), (g + 1) * (hq // h)):
                p = (s["q"][cu[b]:cu[b + 1], i].double() @ k.t()).mul_(s["scale"]).masked_fill_(hide, -math.inf)
                top = p.amax(1, keepdim=True)
                p = p.sub_(torch.where(top.isinf(), torch.zeros_like(top), top)).exp_()
                out[cu[b]:cu[b + 1], i] = (p @ v) / p.sum(1, keepdim=True).clamp_min(1e-300)
    return out
