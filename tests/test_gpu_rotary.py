"""rotary.rotate against the rotation in 64 bits: both layouts, parts of a head, norms, types, strides, gradients, refusals."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def tables(P, R, amp=1.0):
    from statetree_b200.rotary import rotary_tables
    c, s = rotary_tables(R, P, 1e4)
    return c * amp, s * amp


def reference(x, pos, cos, sin, pairs, offset=0, w=None, eps=1e-6, inverse=False):
    """(result in 64 bits, bound on the kernel's error).  The bound: half a step of the type for the one rounding, and 2^-24 of |a| + |b|
    for each of at most sixteen fp32 roundings on the way (norm: a sum of D squares adds D / 32 + 5 of them at most, halved by the root,
    rsqrtf two more; the products and the final sum four)"""
    t, R, D = x.dtype, 2 * cos.shape[1], x.shape[-1]
    y = x.double()
    if w is not None:
        y = y / (y.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
    p = pos.clamp(0, cos.shape[0] - 1).expand(x.shape[0])
    c, s = cos.double()[p][:, None], sin.double()[p][:, None] * (-1 if inverse else 1)
    out, size = y.clone(), y.abs()
    r = y[..., offset:offset + R]
    a, b = (r[..., 0::2], r[..., 1::2]) if pairs else (r[..., :R // 2], r[..., R // 2:])
    u, v = a * c - b * s, a * s + b * c
    m = (a.abs() + b.abs()) * torch.maximum(c.abs(), s.abs())
    put = (lambda z, y0, y1: torch.stack([y0, y1], -1).flatten(-2)) if pairs else (lambda z, y0, y1: torch.cat([y0, y1], -1))
    out[..., offset:offset + R], size[..., offset:offset + R] = put(None, u, v), put(None, m, m)
    f = torch.finfo(t)
    roundings = 16 if w is None else 16 + D // 32
    return out, f.eps / 2 * out.abs() + roundings * 2.0 ** -24 * size * (1 + f.eps) + f.tiny * f.eps / 2


def check(got, x, *args, **kw):
    want, tol = reference(x, *args, **kw)
    assert got.dtype == x.dtype and got.shape == x.shape
    off = (got.double() - want).abs()
    assert bool((off <= tol).all()), float((off / tol).max())


def make(N, H, D, t, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randn(N, H, D, device="cuda", generator=g).to(t)


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("pairs", [True, False])
@pytest.mark.parametrize("D,R,offset", [(128, 128, 0), (64, 64, 0), (80, 32, 0), (96, 48, 48), (256, 64, 16), (192, 64, 128), (512, 512, 0),
                                        (40, 40, 0), (20, 10, 3), (7, 4, 2), (1024, 1024, 0), (16, 0, 0), (48, 16, 8), (2, 2, 0)])
def test_layouts(t, pairs, D, R, offset):
    """whole vectors and odd sizes, first and last parts; q with norm, k without"""
    from statetree_b200.rotary import rotate
    N, Hq, Hk = 13, 5, 3
    q, k = make(N, Hq, D, t), make(N, Hk, D, t, 1)
    w = make(1, 1, D, t, 2)[0, 0] * 0.1 + 1
    cos, sin = tables(50, R) if R else (torch.empty(50, 0, device="cuda"),) * 2
    pos = torch.tensor([0, 49, 7, 3, 3, 60, -4, 12, 1, 2, 48, 30, 20], device="cuda")      # (two outside the table)
    a, b = rotate(q, k, pos, cos, sin, interleaved=pairs, offset=offset, q_norm=w, eps=1e-5)
    check(a, q, pos, cos, sin, pairs, offset, w, 1e-5)
    check(b, k, pos, cos, sin, pairs, offset)
    if offset or R < D:
        keep = torch.ones(D, dtype=torch.bool, device="cuda")
        keep[offset:offset + R] = False
        assert torch.equal(b[..., keep], k[..., keep])


@pytest.mark.parametrize("N", [0, 1, 2, 31, 257, 10000])
@pytest.mark.parametrize("Hq,Hk", [(32, 8), (1, 1), (9, 3), (64, 0), (0, 2)])
def test_token_and_head_counts(N, Hq, Hk):
    from statetree_b200.rotary import rotate
    q, k = make(N, Hq, 128, torch.bfloat16), make(N, Hk, 128, torch.bfloat16, 1)
    cos, sin = tables(300, 128)
    pos = torch.randint(0, 300, (N,), device="cuda", generator=torch.Generator("cuda").manual_seed(3))
    for positions in (pos, torch.tensor([17], device="cuda")):
        a, b = rotate(q, k if Hk else None, positions, cos, sin, interleaved=False)
        check(a, q, positions, cos, sin, False)
        assert b is None if not Hk else check(b, k, positions, cos, sin, False) is None


def test_parts_of_a_fused_row_in_place():
    """q and k as views of q/k/v rows, at an odd element offset and at an aligned one; in place; v stays as it is"""
    from statetree_b200.rotary import rotate
    for shift in (0, 3, 8):
        flat = make(1, 1, 11 * 7 * 64 + 8, torch.bfloat16).view(-1)
        rows = flat[shift:shift + 11 * 7 * 64].view(11, 7, 64)
        q, k, v = rows.split([4, 1, 2], 1)
        before = rows.clone()
        cos, sin = tables(11, 64)
        pos = torch.arange(11, device="cuda")
        a, b = rotate(q, k, pos, cos, sin)
        assert torch.equal(rows, before) and a.is_contiguous()
        c, d = rotate(q, k, pos, cos, sin, out=(q, k))
        assert c is q and d is k and torch.equal(q, a) and torch.equal(k, b) and torch.equal(v, before[:, 5:])
        check(q.clone(), before[:, :4], pos, cos, sin, True)


def test_heads_far_apart_and_shared():
    """strides other than the usual ones: heads in the outer dimension, one head read for several (stride 0), tokens in reverse order"""
    from statetree_b200.rotary import rotate
    x = make(6, 21, 128, torch.bfloat16).transpose(0, 1)                  # [21, 6, 128]: head stride 21 * 128
    k = make(21, 1, 128, torch.bfloat16, 1).expand(21, 4, 128)
    cos, sin = tables(30, 128)
    pos = torch.arange(20, -1, -1, device="cuda")
    a, b = rotate(x, k, pos, cos, sin, interleaved=False)
    check(a, x, pos, cos, sin, False)
    check(b, k, pos, cos, sin, False)


def test_inverse_and_what_is_not_finite():
    """there and back within two roundings; infinities and NaN stay in their pair; values outside the part keep theirs"""
    from statetree_b200.rotary import rotate
    x = make(40, 3, 128, torch.float32)
    cos, sin = tables(64, 64)
    pos = torch.arange(40, device="cuda")
    y, _ = rotate(x, None, pos, cos, sin, offset=32)
    back, _ = rotate(y, None, pos, cos, sin, offset=32, inverse=True)
    m = x.abs()
    m[..., 32:96] = (m[..., 32:96:2] + m[..., 33:96:2]).repeat_interleave(2, -1) * 2
    assert bool(((back - x).abs() <= 16 * 2.0 ** -24 * m).all())
    x[0, 0, 40], x[1, 1, 5] = float("inf"), float("nan")
    z, _ = rotate(x, None, pos, cos, sin, offset=32)
    odd = ~torch.isfinite(z)
    assert odd[0, 0].nonzero().view(-1).tolist() in ([40], [40, 41]) and odd[1, 1].nonzero().view(-1).tolist() == [5]
    assert int(odd.sum()) <= 3
    odd[0, 0, 40:42], odd[1, 1, 5] = True, True
    assert torch.equal(z[~odd], y[~odd])


@pytest.mark.parametrize("t", TYPES, ids=str)
@pytest.mark.parametrize("pairs", [True, False])
def test_gradients(t, pairs):
    """against the formula's (the transposed matrix, with the table's amplitude), from expanded and strided gradients too"""
    from statetree_b200.rotary import rotate
    q, k = make(9, 4, 96, t).requires_grad_(), make(9, 2, 96, t, 1).requires_grad_()
    cos, sin = tables(20, 64, 1.25)
    pos = torch.arange(5, 14, device="cuda")
    a, b = rotate(q, k, pos, cos, sin, interleaved=pairs, offset=32)
    ga, gb = make(9, 4, 96, t, 5), make(4, 9, 96, t, 6)[:2].transpose(0, 1)
    dq, dk = torch.autograd.grad((a, b), (q, k), (ga, gb), retain_graph=True)
    check(dq, ga, pos, cos, sin, pairs, 32, inverse=True)
    check(dk, gb, pos, cos, sin, pairs, 32, inverse=True)
    dq, = torch.autograd.grad(a.sum(), q, retain_graph=True)               # a gradient of stride zero
    check(dq, torch.ones_like(q), pos, cos, sin, pairs, 32, inverse=True)
    dk, = torch.autograd.grad(b, k, gb)                                     # of one output only
    check(dk, gb, pos, cos, sin, pairs, 32, inverse=True)
    a, none = rotate(q, None, pos, cos, sin, interleaved=pairs, offset=32)
    assert none is None
    check(torch.autograd.grad(a, q, ga)[0], ga, pos, cos, sin, pairs, 32, inverse=True)


def test_gradient_against_differences():
    """the function is linear, so a difference of any width is the derivative along its direction: fp32 errors only, 2^-24 of the values
    for each of some 32 roundings, summed over 3 * 64 values"""
    from statetree_b200.rotary import rotate
    x, d, g = make(3, 1, 64, torch.float32).requires_grad_(), make(3, 1, 64, torch.float32, 1), make(3, 1, 64, torch.float32, 2)
    cos, sin = tables(8, 64)
    pos = torch.tensor([1, 7, 3], device="cuda")
    y, _ = rotate(x, None, pos, cos, sin)
    dx, = torch.autograd.grad(y, x, g)
    with torch.no_grad():
        up, down = rotate(x + d, None, pos, cos, sin)[0], rotate(x - d, None, pos, cos, sin)[0]
    slope = ((up.double() - down.double()) / 2 * g.double()).sum()
    bound = 32 * 2.0 ** -24 * float(((x.detach().abs() + d.abs()).double() * 2 * g.abs().double()).sum() + (dx.abs() * d.abs()).double().sum())
    assert abs(float(slope - (dx.double() * d.double()).sum())) <= bound


def test_gradient_of_a_gradient():
    from statetree_b200.rotary import rotate
    x = make(3, 2, 64, torch.float32).requires_grad_()
    cos, sin = tables(8, 64)
    pos = torch.arange(3, device="cuda")
    g = make(3, 2, 64, torch.float32, 1).requires_grad_()
    dx, = torch.autograd.grad(rotate(x, None, pos, cos, sin)[0], x, g, create_graph=True)
    h = make(3, 2, 64, torch.float32, 2)
    dg, = torch.autograd.grad(dx, g, h)
    check(dg, h, pos, cos, sin, True)


def test_graph_streams_and_replay():
    """captured and replayed over new inputs and positions; on a side stream; the two do not meet"""
    from statetree_b200.rotary import rotate
    q, k, pos = make(17, 4, 128, torch.bfloat16), make(17, 2, 128, torch.bfloat16, 1), torch.arange(17, device="cuda")
    cos, sin = tables(40, 128)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        rotate(q, k, pos, cos, sin)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            a, b = rotate(q, k, pos, cos, sin)
    torch.cuda.current_stream().wait_stream(side)
    for seed in (3, 4):
        q.copy_(make(17, 4, 128, torch.bfloat16, seed))
        pos.copy_(torch.arange(17, device="cuda") + seed)
        graph.replay()
        check(a, q, pos, cos, sin, True)
        check(b, k, pos, cos, sin, True)


def test_far_memory():
    """values beyond 2^31 of a buffer: offsets are formed in 64 bits"""
    from statetree_b200.rotary import rotate
    if torch.cuda.mem_get_info()[0] < 24 << 30:
        pytest.skip("needs 24 GB")
    rows = torch.zeros((1 << 31) + (1 << 20), dtype=torch.bfloat16, device="cuda")
    x = rows.as_strided((2, 2, 128), ((1 << 31), 1 << 14, 1))
    x.copy_(make(2, 2, 128, torch.bfloat16))
    cos, sin = tables(4, 128)
    pos = torch.tensor([3, 1], device="cuda")
    a, _ = rotate(x, None, pos, cos, sin)
    check(a, x, pos, cos, sin, True)
    want = a.clone()
    rotate(x, None, pos, cos, sin, out=(x, None))
    assert torch.equal(x, want)


def test_refusals():
    from statetree_b200.rotary import rotate
    q, k = make(4, 2, 64, torch.bfloat16), make(4, 1, 64, torch.bfloat16)
    cos, sin = tables(8, 64)
    pos = torch.arange(4, device="cuda")
    w = torch.ones(64, dtype=torch.bfloat16, device="cuda")
    far = dict(args=(q, k, pos, cos, sin))
    assert rotate(*far["args"])[0].shape == q.shape
    bad = [((q, k.float(), pos, cos, sin), {}), ((q, k[:3], pos, cos, sin), {}), ((q, k, pos.int(), cos, sin), {}), ((q, k, pos[:3], cos, sin), {}),
           ((q, k, pos, cos.double(), sin.double()), {}), ((q, k, pos, cos, sin[:4]), {}), ((q, k, pos, cos[:0], sin[:0]), {}),
           ((q, k, pos, cos, sin), dict(offset=2)), ((q, k, pos, cos, sin), dict(offset=-1)), ((q, k, pos, cos, sin), dict(q_norm=w[:32])),
           ((q, k, pos, cos, sin), dict(k_norm=w.float())), ((q, k, pos.cpu(), cos, sin), {}), ((q, k, pos, cos.cpu(), sin.cpu()), {}),
           ((q.transpose(1, 2), None, pos, cos, sin), {}), ((q.to(torch.float64), None, pos, cos, sin), {}), ((q[0], None, pos, cos, sin), {}),
           ((q, k, pos, cos, sin), dict(out=(q[:, :1].expand(4, 2, 64), k))), ((q, k, pos, cos, sin), dict(out=(k.expand(4, 2, 64), k))),
           ((q, q[:, 1:], pos, cos, sin), dict(out=(q, torch.empty_like(k)))), ((q, k, pos, cos, sin), dict(out=(torch.empty_like(q), q[:, :1]))),
           ((q, None, pos, cos, sin), dict(out=(q.float(), None)))]
    for args, kw in bad:
        before = q.clone(), k.clone()
        with pytest.raises(RuntimeError):
            rotate(*args, **kw)
        assert torch.equal(q, before[0]) and torch.equal(k, before[1])
    with pytest.raises(RuntimeError, match="gradients"):
        rotate(q.clone().requires_grad_(), k, pos, cos, sin, k_norm=w)


@pytest.mark.parametrize("t", TYPES)
@pytest.mark.parametrize("N,D", [(1, 64), (2, 64), (37, 64), (37, 80), (130, 128)])
def test_heads_outside_tokens_in_place(t, N, D):
    """memory [heads, tokens, D], as attention modules hold it, rotated in place"""
    from statetree_b200.rotary import rotate
    q, k = (make(H, N, D, t).transpose(0, 1) for H in (5, 2))
    before = q.clone(), k.clone()
    cos, sin = tables(N, 64)
    pos = torch.arange(N, device="cuda")
    want = rotate(*before, pos, cos, sin)
    got = rotate(q, k, pos, cos, sin, out=(q, k))
    assert got[0] is q and got[1] is k and torch.equal(q, want[0]) and torch.equal(k, want[1])
    both = make(7, N, D, t)                                  # (q and k beside one another in one buffer)
    q, k = both[:5].transpose(0, 1), both[5:].transpose(0, 1)
    want = rotate(q.clone(), k.clone(), pos, cos, sin)
    rotate(q, k, pos, cos, sin, out=(q, k))
    assert torch.equal(q, want[0]) and torch.equal(k, want[1])
