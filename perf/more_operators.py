"""A decoder layer on a chunk of prompt tokens as measurable cases: what it needs beside a decode step when weights are state trees and
the cache is lossless pages.

`kind` names the operator:

  rotary  queries and keys rotated by their tokens' positions, in either layout, whole heads or a part of each, with the per-head
          RMSNorm in front (`norm`) or, for training, with the gradients (`train`)
  chunk   causal attention of up to `new` query tokens per sequence that stand at the end of up to `ctx` cached ones, over the pages
  linear  act(x W^T + bias) + residual for a state-tree weight W of `out` x `cols`; act "swiglu": W holds gate and up in 16-row tiles in
          turn, and the result is silu(gate x) * (up x)

A page holds 16 tokens of one layer, uint8 [blocks, KV heads, 2 (keys, values), 2 (halves of the head), 1600].  A unit of 1600 bytes is
16 rows x 64 values: leaves (mantissa << 1 | sign of the neighbour), four-bit states (how far a value's exponent is below its row's
largest), the rows' largest exponents, a header word and eleven entries for the exact bits of values that lie more than 14 exponents
below; further entries chain through 64-byte blocks of a pool.

Lengths depend on the case alone (`ragged`: spread over the range, some sequences without tokens), values on the seed.
"""
import math
import os
import sys

import torch

own = False
DEV = "cuda"
PAGE, UNIT, D = 16, 1600, 128                # (heads of the pages)
HEADER, SLOTS, EXTRA = 1552, 11, 15
TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}


def listed():
    return [
        # a decode step of one user: the smallest call, latency counts
        dict(name="rotary_step_b1", kind="rotary", tokens=1, far=4000, heads=32, kv_heads=8, dim=128, part=128, pairs=True, norm=True,
             type="bf16", scaled="none", train=False),
        # half of a wider head rotated, odd number of tokens, half precision
        dict(name="rotary_part_d80", kind="rotary", tokens=1261, far=20000, heads=32, kv_heads=32, dim=80, part=32, pairs=False, norm=False,
             type="f16", scaled="linear", train=False),
        # a training batch: forward and both gradients
        dict(name="rotary_train_8k", kind="rotary", tokens=8190, far=0, heads=16, kv_heads=16, dim=128, part=128, pairs=False, norm=False,
             type="bf16", scaled="none", train=True),
        # long prompts at far positions of a context that was stretched
        dict(name="rotary_prompt_32k", kind="rotary", tokens=32764, far=90000, heads=32, kv_heads=8, dim=128, part=128, pairs=False, norm=True,
             type="bf16", scaled="yarn", train=False),
        # speculative tokens of a few users
        dict(name="chunk_b8_t4", kind="chunk", seqs=8, new=4, ctx=2900, ragged=False, heads=32, kv_heads=8, window=0, pad=0),
        # chunks of different lengths over different contexts, a sliding window, left padding, seven query heads per KV head
        dict(name="chunk_ragged_window", kind="chunk", seqs=9, new=700, ctx=2500, ragged=True, heads=28, kv_heads=4, window=900, pad=33),
        # a prompt from its beginning
        dict(name="chunk_prompt_4k", kind="chunk", seqs=1, new=4096, ctx=0, ragged=False, heads=32, kv_heads=8, window=0, pad=0),
        # a late chunk of a very long prompt
        dict(name="chunk_2k_over_30k", kind="chunk", seqs=1, new=2048, ctx=30000, ragged=False, heads=32, kv_heads=8, window=0, pad=0),
        # a decode step's down projection, added to the residual stream
        dict(name="linear_b1_residual", kind="linear", rows=1, out=4096, cols=12288, act="none", bias=False, residual=True),
        # a small layer with bias and activation, rows that fill no tile on either side
        dict(name="linear_b37_gelu", kind="linear", rows=37, out=4304, cols=1152, act="gelu", bias=True, residual=False),
        # gate and up of a short prompt
        dict(name="linear_b300_swiglu", kind="linear", rows=300, out=24576, cols=4096, act="swiglu", bias=False, residual=False),
        # a long chunk's down projection, added to the residual stream
        dict(name="linear_b2000_residual", kind="linear", rows=2000, out=4096, cols=12288, act="none", bias=True, residual=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))


def draw(rng):
    kind = rng.choice(("rotary", "chunk", "linear"))
    if kind == "rotary":
        heads, kv = rng.choice(((32, 8), (28, 4), (16, 16), (8, 1), (14, 2), (9, 3), (64, 8)))
        dim = rng.choice((64, 80, 96, 128, 192, 256))
        part = rng.choice((dim, dim, dim // 2, 32))
        train = rng.random() < 0.3
        return dict(kind=kind, tokens=_log(rng, 1, 32768 * 40 * 128 // ((heads + kv) * dim * (2 if train else 1))), far=rng.choice((0, 500, 120000)),
                    heads=heads, kv_heads=kv, dim=dim, part=part, pairs=rng.random() < 0.5, norm=not train and rng.random() < 0.5,
                    type=rng.choice(("bf16", "bf16", "f16", "f32")), scaled=rng.choice(("none", "linear", "yarn")), train=train)
    if kind == "chunk":
        heads, kv = rng.choice(((32, 8), (28, 4), (16, 16), (8, 1), (40, 8), (12, 1), (9, 3), (64, 4)))
        seqs = _log(rng, 1, 24)
        new = _log(rng, 1, 4096 // seqs)
        return dict(kind=kind, seqs=seqs, new=new, ctx=_log(rng, 1, min(32768, (1 << 30) // (seqs * new * heads) + 16, 262144 // seqs)),
                    ragged=rng.random() < 0.6, heads=heads, kv_heads=kv, window=rng.choice((0, 0, 0, 1, 100, 777, 4096)),
                    pad=rng.choice((0, 0, 5, 200)))
    act = rng.choice(("none", "none", "relu", "silu", "gelu", "gelu_tanh", "swiglu"))
    step = 128 if act == "swiglu" else 16
    cols = 64 * _log(rng, 1, 192)
    out = step * _log(rng, 1, min(24576, (24576 * 4096) // cols) // step)
    return dict(kind=kind, rows=_log(rng, 1, min(4096, 2000 * 4096 * 12288 // (out * cols))), out=out, cols=cols, act=act,
                bias=rng.random() < 0.5, residual=act != "swiglu" and rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ lengths, work
def _spread(c, hi, salt):
    """a length per sequence: all `hi`, or spread over [0, hi] by the golden ratio, the first one `hi`"""
    if not c["ragged"]:
        return [hi] * c["seqs"]
    return [hi if b == 0 else int((b * 0.6180339887498949 + salt) % 1.0 * (hi + 1)) for b in range(c["seqs"])]


def _chunk_lens(c):
    """(new tokens, tokens in all, first token that takes part) per sequence"""
    new, old = _spread(c, c["new"], 0.1), _spread(c, c["ctx"], 0.5)
    lens = [n + o for n, o in zip(new, old)]
    return new, lens, [min(n, c["pad"] * (b % 2)) for b, n in enumerate(lens)]


def work(case):
    c = case
    if c["kind"] == "rotary":
        n, size = c["tokens"], 4 if c["type"] == "f32" else 2
        values = n * (c["heads"] + c["kv_heads"]) * c["dim"] * (2 if c["train"] else 1)
        return dict(bytes=2 * values * size + n * (8 + 4 * c["part"]), flops=6 * values)
    if c["kind"] == "linear":
        b, m, n = c["rows"], c["out"], c["cols"]
        y = m // 2 if c["act"] == "swiglu" else m
        return dict(bytes=m * n // 1024 * 1552 + 2 * b * (n + y * (2 if c["residual"] else 1)), flops=2 * b * m * n)
    new, lens, starts = _chunk_lens(c)
    win = c["window"] or 1 << 60
    seen = cached = 0
    for n, m, s in zip(new, lens, starts):
        seen += sum(max(0, p + 1 - max(s, p + 1 - win)) for p in range(m - n, m))
        cached += max(0, m - max(s, m - n + 1 - win)) if n else 0
    return dict(bytes=cached * c["kv_heads"] * 4 * UNIT // PAGE + 4 * sum(new) * c["heads"] * D, flops=4 * D * c["heads"] * seen)


# ------------------------------------------------------------------------------------------------ pages
def _encode(x, pool_from):
    """BF16 x [pages, 16, heads, 128] of keys or values -> (units uint8 [pages, heads, 2, 1600], pool blocks int32 [n, 16] that follow
    block pool_from - 1, longest chain)"""
    P, _, H, _ = x.shape
    v = x.view(torch.int16).int() & 0xFFFF
    v = v.view(P, PAGE, H, 2, 64).permute(0, 2, 3, 1, 4).reshape(-1, PAGE, 64)                # [unit, row, column]
    U = v.shape[0]
    e = v >> 7 & 255
    top = e.amax(-1, keepdim=True)
    out = top - e > 14
    sign = torch.where(out, 0, v >> 15).view(U, PAGE, 32, 2).flip(-1).reshape(U, PAGE, 64)    # (kept beside the neighbour)
    leaf = (torch.where(out, 0, (v & 127) << 1) | sign).to(torch.uint8)
    state = torch.where(out, 15, top - e).to(torch.uint8)
    units = torch.zeros(U, UNIT, dtype=torch.uint8, device=x.device)
    # column = 16 s + 8 i + 2 t + b, row = 8 j + r
    units[:, :1024] = leaf.view(U, 2, 8, 2, 2, 2, 4, 2).permute(0, 3, 2, 6, 4, 1, 5, 7).reshape(U, 1024)
    q = state.view(U, 2, 8, 4, 2, 4, 2)
    units[:, 1024:1536] = (q[:, 0] | q[:, 1] << 4).permute(0, 1, 4, 2, 3, 5).reshape(U, 512)
    units[:, 1536:1552] = top.view(U, 2, 8).transpose(1, 2).reshape(U, 16).to(torch.uint8)
    unit, row, col = out.nonzero(as_tuple=True)                                               # row by row, column by column
    entry = (v[unit, row, col] << 16 | row.int() << 6 | col.int())
    count = torch.bincount(unit, minlength=U)
    rank = torch.arange(unit.numel(), device=x.device) - (count.cumsum(0) - count)[unit]
    words = units.view(torch.int32)                                                           # [unit, 400]
    here = rank < SLOTS
    words[unit[here], HEADER // 4 + 1 + rank[here]] = entry[here]
    blocks = ((count - SLOTS).clamp_min(0) + EXTRA - 1) // EXTRA
    first = blocks.cumsum(0) - blocks + pool_from
    words[:, HEADER // 4] = torch.where(blocks > 0, first << 8 | 16, 0).int() | count.clamp_max(SLOTS).int()
    n = int(blocks.sum())
    pool = torch.zeros(n, 16, dtype=torch.int32, device=x.device)
    if n:
        far = ~here
        at = (rank[far] - SLOTS)
        blk = first[unit[far]] - pool_from + at // EXTRA
        pool[blk, 1 + at % EXTRA] = entry[far]
        owner = torch.repeat_interleave(torch.arange(U, device=x.device), blocks)
        i = torch.arange(n, device=x.device) - (first - pool_from)[owner]
        last = i + 1 == blocks[owner]
        used = torch.where(last, (count - SLOTS)[owner] - i * EXTRA, EXTRA)
        pool[:, 0] = (used + torch.where(last, 0, (torch.arange(n, device=x.device) + pool_from + 2) << 8)).int()
    return units.view(P, H, 2, UNIT), pool, int(blocks.max())


def _decode(units, pool, hops):
    """units uint8 [n, 1600] -> the float32 values [n, 16, 64] that they stand for"""
    U = units.shape[0]
    leaf = units[:, :1024].view(U, 2, 8, 4, 2, 2, 2, 2).permute(0, 5, 2, 1, 4, 6, 3, 7).reshape(U, PAGE, 64).int()
    q = units[:, 1024:1536].view(U, 8, 4, 4, 2, 2).permute(0, 1, 3, 4, 2, 5).reshape(U, 1, 8, 64).int()
    state = torch.cat([q & 15, q >> 4], 1).view(U, PAGE, 64)
    top = units[:, 1536:1552].view(U, 8, 2).transpose(1, 2).reshape(U, PAGE, 1).int()
    sign = (leaf & 1).view(U, PAGE, 32, 2).flip(-1).reshape(U, PAGE, 64)
    bits = (sign << 15 | (top - state) << 7 | leaf >> 1).view(U, PAGE * 64)
    words = units.view(torch.int32)
    head = words[:, HEADER // 4]
    bits = torch.cat([bits, bits[:, :1]], 1)                                                  # (a column for entries that are none)
    put = lambda e, live: bits.scatter_(1, torch.where(live, (e & 1023).long(), PAGE * 64), e >> 16 & 0xFFFF)     # noqa: E731
    put(words[:, HEADER // 4 + 1:HEADER // 4 + 1 + SLOTS], torch.arange(SLOTS, device=units.device) < (head & 15)[:, None])
    if hops:
        block = torch.where(head & 16 > 0, head >> 8, -1)
        for _ in range(hops):
            b = pool[block.clamp_min(0).long()]
            put(b[:, 1:], (torch.arange(EXTRA, device=units.device) < (b[:, 0] & 255)[:, None]) & (block >= 0)[:, None])
            block = torch.where(block >= 0, (b[:, 0] >> 8) - 1, -1)
    return (bits[:, :-1] << 16).view(torch.float32).view(U, PAGE, 64)


# ------------------------------------------------------------------------------------------------ inputs
def _package():
    pkg = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "statetree-representation_b200")
    if pkg not in sys.path:
        sys.path.insert(0, pkg)


def _frequencies(c):
    """(angle per position of every pair in 64 bits, factor of the table) after the kind of scaling"""
    R, theta = c["part"], 5e5
    inv = theta ** (-torch.arange(0, R, 2, device=DEV, dtype=torch.float64) / R)
    if c["scaled"] == "linear":
        return inv / 4.0, 1.0
    if c["scaled"] == "yarn":                                # pairs that turn often keep their speed, slow ones are stretched
        factor, trained, fast, slow = 8.0, 16384, 32.0, 1.0
        at = lambda turns: R * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))          # noqa: E731
        lo, hi = max(0, math.floor(at(fast))), min(R - 1, math.ceil(at(slow)))
        ramp = ((torch.arange(R // 2, device=DEV, dtype=torch.float64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        return inv * (1 - ramp) + inv / factor * ramp, 0.1 * math.log(factor) + 1.0
    return inv, 1.0


def prepare(case, seed):
    c = case
    gen = torch.Generator(device=DEV).manual_seed(1 + int(seed))
    rand = lambda *shape: torch.randn(*shape, device=DEV, generator=gen)                      # noqa: E731
    ints = lambda v, t=torch.int32: torch.tensor(v, dtype=t, device=DEV)                      # noqa: E731
    if own:
        _package()
    if c["kind"] == "rotary":
        n, hq, h, d, t = c["tokens"], c["heads"], c["kv_heads"], c["dim"], TYPES[c["type"]]
        inv, factor = _frequencies(c)
        ang = torch.arange(c["far"] + n, device=DEV, dtype=torch.float64)[:, None] * inv
        state = dict(case=c, cos=(ang.cos() * factor).float(), sin=(ang.sin() * factor).float(),
                     positions=c["far"] + torch.randperm(n, device=DEV, generator=gen))       # (tokens of several sequences)
        if c["train"]:
            q, k = rand(n, hq, d).to(t), rand(n, h, d).to(t)
            return dict(state, q=q.requires_grad_(own), k=k.requires_grad_(own), dq=rand(n, hq, d).to(t), dk=rand(n, h, d).to(t))
        rows = rand(n, hq + 2 * h, d).to(t)                                                   # queries, keys and values as a projection leaves them
        q, k, _ = rows.split([hq, h, h], 1)
        w = [(1 + 0.1 * rand(d)).to(t) if c["norm"] else None for _ in range(2)]
        return dict(state, q=q, k=k, wq=w[0], wk=w[1])
    if c["kind"] == "linear":
        m, n, b = c["out"], c["cols"], c["rows"]
        W = rand(m, n) * 0.02
        W[:, torch.randperm(n, device=DEV, generator=gen)[:max(1, n // 100)]] *= 8
        W = W.to(torch.bfloat16)
        bias = rand(m).to(torch.bfloat16) if c["bias"] else None
        state = dict(case=c, x=rand(b, n).to(torch.bfloat16), residual=rand(b, m).to(torch.bfloat16) * 3 if c["residual"] else None)
        if own:
            from statetree_b200 import TreeLinear
            return dict(state, layer=TreeLinear.from_weight(W, bias, verify=False))
        return dict(state, W=W, bias=bias)
    new, lens, starts = _chunk_lens(c)
    h, hq = c["kv_heads"], c["heads"]
    width = max(1, -(-max(lens) // PAGE))
    pages = c["seqs"] * width
    kv = torch.empty(pages, h, 2, 2, UNIT, dtype=torch.uint8, device=DEV)
    size = rand(h, D).exp()                                                                   # channels of different sizes
    size[0, 5] = 1e-6                                                                         # ... and one that is nearly dead
    pools, hops, have = [], 0, 0
    step = max(1, (1 << 25) // (PAGE * h * D))
    for p in range(0, pages, step):                                                           # (a large cache is filled in parts)
        shape = (min(step, pages - p), PAGE, h, D)
        for i, x in enumerate((rand(*shape) * size, rand(*shape))):
            kv[p:p + step, :, i], pool, most = _encode(x.to(torch.bfloat16), have)
            pools.append(pool)
            have, hops = have + pool.shape[0], max(hops, most)
    pool = torch.cat(pools + [torch.zeros(64, 16, dtype=torch.int32, device=DEV)])
    state = dict(case=c, pages=kv, pool=pool, hops=hops, q=(rand(sum(new), hq, D) * 1.5).to(torch.bfloat16), lens=ints(lens), scale=D ** -0.5,
                 table=torch.randperm(pages, device=DEV, generator=gen).to(torch.int32).view(c["seqs"], width),
                 cu=ints([sum(new[:b]) for b in range(c["seqs"] + 1)]), longest=max(new), starts=ints(starts) if c["pad"] else None)
    if own:
        from statetree_b200.kvcache import PageStore
        state["store"] = PageStore.over(kv, pool)
    return state


# ------------------------------------------------------------------------------------------------ one pass
def _rotated(x, w, cos, sin, c):
    """x [tokens, heads, dim] in its type: RMSNorm with weights w (None: none), then the rotation of the first `part` values"""
    y = x.float()
    if w is not None:
        y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + 1e-6) * w.float()
    r, rest = y[..., :c["part"]], y[..., c["part"]:]
    a, b = (r[..., 0::2], r[..., 1::2]) if c["pairs"] else r.chunk(2, -1)
    z = a * cos - b * sin, a * sin + b * cos
    return torch.cat([torch.stack(z, -1).flatten(-2) if c["pairs"] else torch.cat(z, -1), rest], -1).to(x.dtype)


def _rotary(s):
    c = s["case"]
    if own:
        from statetree_b200.rotary import rotate
        if not c["train"]:
            q, k = rotate(s["q"], s["k"], s["positions"], s["cos"], s["sin"], interleaved=c["pairs"], q_norm=s["wq"], k_norm=s["wk"], eps=1e-6)
            return dict(q=q, k=k)
        q, k = rotate(s["q"], s["k"], s["positions"], s["cos"], s["sin"], interleaved=c["pairs"])
        gq, gk = torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"]))
        return dict(q=q.detach(), k=k.detach(), gq=gq, gk=gk)
    cos, sin = s["cos"][s["positions"]][:, None], s["sin"][s["positions"]][:, None]
    out = dict(q=_rotated(s["q"], s.get("wq"), cos, sin, c), k=_rotated(s["k"], s.get("wk"), cos, sin, c))
    if c["train"]:                                           # the gradient is the rotation by the opposite angle
        out.update(gq=_rotated(s["dq"], None, cos, -sin, c), gk=_rotated(s["dk"], None, cos, -sin, c))
    return out


_ACTS = {"none": lambda z: z, "relu": lambda z: z.clamp_min(0), "silu": lambda z: z / (1 + (-z).exp()),
         "gelu": lambda z: 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5))),
         "gelu_tanh": lambda z: 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))}


def _linear(s):
    act = s["case"]["act"]
    if own:
        return s["layer"].fused(s["x"], activation=None if act == "none" else act, residual=s["residual"])
    z = torch.matmul(s["x"].float(), s["W"].float().t())
    if s["bias"] is not None:
        z = z + s["bias"].float()
    if act == "swiglu":
        g = z.view(z.shape[0], -1, 2, 16)
        y = (_ACTS["silu"](g[:, :, 0]) * g[:, :, 1]).flatten(1)
    else:
        y = _ACTS[act](z)
    if s["residual"] is not None:
        y = y + s["residual"].float()
    return y.to(torch.bfloat16)


def _chunk(s):
    c = s["case"]
    if own:
        return s["store"].chunk_attention(s["q"], s["cu"], s["table"], s["lens"], s["scale"], starts=s["starts"], window=c["window"])
    new = s["cu"][1:] - s["cu"][:-1]
    i = torch.arange(s["longest"], device=DEV)
    live = i[None] < new[:, None]                                                             # rows of the padded batch that are queries
    row = (s["cu"][:-1, None] + i).clamp_max(s["q"].shape[0] - 1)
    at = torch.where(live, (s["lens"] - new)[:, None] + i, -1)
    q = s["q"][row.long()].float()                                                            # [seqs, longest, heads, dim]
    B, n, hq, _ = q.shape
    h, width = c["kv_heads"], s["table"].shape[1]
    x = _decode(s["pages"][s["table"].long()].view(-1, UNIT), s["pool"], s["hops"]).view(B, width, h, 2, 2, PAGE, 64)
    k, v = (x[:, :, :, j].permute(0, 2, 1, 4, 3, 5).reshape(B, h, width * PAGE, D) for j in range(2))
    del x
    S = torch.matmul(q.view(B, n, h, hq // h, D).permute(0, 2, 1, 3, 4).reshape(B, h, n * (hq // h), D) * s["scale"], k.transpose(2, 3))
    j = torch.arange(width * PAGE, device=DEV)
    seen = j <= at[..., None]
    if s["starts"] is not None:
        seen &= j >= s["starts"][:, None, None]
    if c["window"]:
        seen &= j > at[..., None] - c["window"]
    S = S.view(B, h, n, hq // h, -1).masked_fill_(~seen[:, None, :, None], float("-inf")).view(S.shape)
    top = S.amax(-1, keepdim=True).clamp_min(-3e38)                                           # (a row that sees nothing: sums of zero)
    P = S.sub_(top).exp_()
    o = (torch.matmul(P, v) / P.sum(-1, keepdim=True).clamp_min(1e-30)).view(B, h, n, hq // h, D).permute(0, 2, 1, 3, 4).reshape(B, n, hq, D)
    token = torch.arange(s["q"].shape[0], device=DEV)
    seq = torch.searchsorted(s["cu"][1:], token.int(), right=True)
    return o[seq, token - s["cu"][seq]].to(torch.bfloat16)


def run(state):
    kind = state["case"]["kind"]
    return _rotary(state) if kind == "rotary" else _linear(state) if kind == "linear" else _chunk(state)


# ------------------------------------------------------------------------------------------------ in 64 bits
def _exact_rotary(c, s):
    inv, factor = _frequencies(c)
    R = c["part"]
    turn = torch.polar(torch.full((c["tokens"], R // 2), factor, dtype=torch.float64, device=DEV), s["positions"].double()[:, None] * inv)[:, None]

    def rot(x, w, by):
        x = x.double()
        if w is not None:
            x = x / (x.pow(2).sum(-1, keepdim=True) / c["dim"] + 1e-6).sqrt() * w.double()
        r = x[..., :R]
        z = torch.view_as_complex(r.reshape(*r.shape[:-1], R // 2, 2).contiguous() if c["pairs"] else
                                  r.reshape(*r.shape[:-1], 2, R // 2).transpose(-1, -2).contiguous()) * by
        z = torch.view_as_real(z)
        return torch.cat([(z if c["pairs"] else z.transpose(-1, -2)).reshape(r.shape), x[..., R:]], -1)

    with torch.no_grad():
        out = dict(q=rot(s["q"], s.get("wq"), turn), k=rot(s["k"], s.get("wk"), turn))
        if c["train"]:
            out.update(gq=rot(s["dq"], None, turn.conj()), gk=rot(s["dk"], None, turn.conj()))
    return out


def _exact_linear(c, s):
    z = s["x"].double() @ s["W"].double().t() + (0 if s["bias"] is None else s["bias"].double())
    if c["act"] == "swiglu":
        gate, up = z.view(z.shape[0], -1, 32).split(16, -1)
        z = (gate * torch.sigmoid(gate) * up).flatten(1)
    elif c["act"] == "relu":
        z = torch.where(z > 0, z, 0)
    elif c["act"] == "silu":
        z = z * torch.sigmoid(z)
    elif c["act"] == "gelu":
        z = z * (0.5 * torch.erfc(-z / math.sqrt(2)))
    elif c["act"] == "gelu_tanh":
        z = z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z if s["residual"] is None else z + s["residual"].double()


def _exact_chunk(c, s):
    hq, h = c["heads"], c["kv_heads"]
    lens, cu = s["lens"].tolist(), s["cu"].tolist()
    starts = s["starts"].tolist() if s["starts"] is not None else [0] * c["seqs"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV)
    for b, (m, first) in enumerate(zip(lens, starts)):
        n = cu[b + 1] - cu[b]
        if n == 0:
            continue
        at = torch.arange(m - n, m, device=DEV)[:, None]
        j = torch.arange(m, device=DEV)[None]
        hide = (j > at) | (j < first) | ((j <= at - c["window"]) if c["window"] else j < 0)
        units = s["pages"][s["table"][b, :-(-m // PAGE)].long()]                              # [pages, heads, 2, 2, 1600]
        for g in range(h):
            k, v = (torch.cat([_values(units[:, g, i, half], s["pool"]) for half in range(2)], -1)[:m] for i in range(2))
            for i in range(g * (hq // h), (g + 1) * (hq // h)):
                p = (s["q"][cu[b]:cu[b + 1], i].double() @ k.t()).mul_(s["scale"]).masked_fill_(hide, -math.inf)
                top = p.amax(1, keepdim=True)
                p = p.sub_(torch.where(top.isinf(), torch.zeros_like(top), top)).exp_()
                out[cu[b]:cu[b + 1], i] = (p @ v) / p.sum(1, keepdim=True).clamp_min(1e-300)
    return out


def _values(units, pool):
    """units uint8 [n, 1600] -> float64 [n * 16, 64]: every value found by its byte's place"""
    r, col = torch.arange(PAGE, device=DEV)[:, None], torch.arange(64, device=DEV)[None]
    s, i, t, b = col // 16, col // 8 % 2, col % 8 // 2, col % 2
    at = s // 2 * 512 + (r % 8 * 4 + t) * 16 + (s % 2 * 2 + r // 8) * 4 + 2 * i
    leaf, other = units[:, at + b].double(), units[:, at + 1 - b].double()
    state = torch.div(units[:, 1024 + (r % 8 * 4 + t) * 16 + s * 4 + 2 * i + b], 16 ** (r // 8), rounding_mode="floor").double() % 16
    e = units[:, 1536 + 2 * (r % 8) + r // 8].double() - state
    mant = torch.floor(leaf / 2)
    x = torch.where(e > 0, (1 + mant / 128) * torch.exp2(e - 127), mant * 2.0 ** -133) * (1 - 2 * (other % 2))
    word = units.contiguous().view(torch.int32)
    n = word[:, HEADER // 4]
    lists = [(torch.arange(units.shape[0], device=DEV), word[:, HEADER // 4 + 1:HEADER // 4 + 1 + SLOTS], n % 16)]
    who, blk = (n & 16 > 0).nonzero()[:, 0], None
    blk = n[who] >> 8
    while who.numel():
        row = pool[blk.long()]
        lists.append((who, row[:, 1:], row[:, 0] & 255))
        more = row[:, 0] >> 8 > 0
        who, blk = who[more], (row[more, 0] >> 8) - 1
    for owner, entries, used in lists:
        u, k = (torch.arange(entries.shape[1], device=DEV)[None] < used[:, None]).nonzero(as_tuple=True)
        bits = entries[u, k]
        x[owner[u], (bits >> 6 & 15).long(), (bits & 63).long()] = (bits >> 16).to(torch.int16).view(torch.bfloat16).double()
    return x.reshape(-1, 64)


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotary": _exact_rotary, "linear": _exact_linear, "chunk": _exact_chunk}[case["kind"]](case, s)
