"""Rotary positions: the tables of a model's position encoding and the rotation of many tokens' queries and keys by them (a decode
step's is fused into its append: ops.kv_ext().rope_append, PageStore8.append).  No counterpart in the reference, whose models bring
their own modules.

    cos, sin = rotary_tables(128, 131072, theta=5e5, scaling=dict(rope_type="llama3", factor=8.0, original_max_position_embeddings=8192))
    q, k = rotate(q, k, positions, cos, sin, interleaved=False)
"""
import math

import torch
import torch.autograd.forward_ad as forward_ad

from .ops import calls, ext


# what rotary_tables reads of a configuration's rope_scaling: of every kind, of its own.  (partial_rotary_factor is in `part`; a model's and its
# trained length are looked at by the kinds that need them)
_KEYS = {"rope_type", "type", "rope_theta", "partial_rotary_factor", "original_max_position_embeddings", "max_position_embeddings"}
_KIND_KEYS = {"default": set(), "linear": {"factor"}, "dynamic": {"factor"},
              "yarn": {"factor", "beta_fast", "beta_slow", "truncate", "attention_factor", "mscale", "mscale_all_dim"},
              "llama3": {"factor", "low_freq_factor", "high_freq_factor"}, "longrope": {"factor", "attention_factor", "short_factor", "long_factor"}}


def rotary_tables(part, length, theta=None, scaling=None, device="cuda"):
    """(cos, sin) float32 [length, part / 2] for positions 0 .. length - 1: angle position * theta^(-2i / part), formed in 64 bits (a far
    position times a rounded frequency is off by whole radians in 32).  theta: by default scaling's rope_theta (where a configuration
    keeps it there), else 10000; two that differ are refused.  scaling: a model configuration's rope_scaling, a dict with rope_type (or type)
    and the keys of its kind; a key with a value that its kind does not read is refused, since a model that reads it has another table (one
    dict per kind of layer: pass the layer's).  `part` is the head's dimension times the configuration's partial_rotary_factor

      default   none
      linear    factor: positions are divided by it
      dynamic   factor, max_position_embeddings (without it original_max_position_embeddings): theta grows once `length` is beyond that
                length, so that the slowest pair's angle grows by factor * length / trained - factor + 1 less
      yarn      factor, original_max_position_embeddings [, beta_fast 32, beta_slow 1, truncate True, attention_factor]: pairs that turn
                more than beta_fast times over the trained length keep their speed, those below beta_slow are divided by factor, a
                line between, which begins and ends at whole pairs (truncate false: where the turns say); cos and sin times
                attention_factor (0.1 ln(factor) + 1; with mscale m and mscale_all_dim a both given and not 0, (0.1 m ln(factor) + 1) /
                (0.1 a ln(factor) + 1))
      llama3    factor, original_max_position_embeddings, low_freq_factor 1, high_freq_factor 4: the same by wavelength
      longrope  short_factor / long_factor (one number a pair; the long ones beyond the trained length), original_max_position_embeddings:
                every pair divided by its own; cos and sin times attention_factor, by default sqrt(1 + ln(s) / ln(trained length)) for
                a stretch s above 1, which is factor or, without one, max_position_embeddings / original_max_position_embeddings.
                The stretch is the model's, whatever the `length` of a table: one of the three must be given (a configuration
                keeps max_position_embeddings beside its rope_scaling: dict(rope_scaling, max_position_embeddings=...))"""
    if part < 2 or part % 2 or length < 1:
        raise ValueError(f"rotary_tables: an even number of values and at least one position, got {part} and {length}")
    sc = dict(scaling or {})
    known = sc.get("rope_theta")
    if theta is not None and known is not None and float(theta) != float(known):
        raise ValueError(f"rotary_tables: theta {theta}, and rope_theta {known} in the scaling")
    theta = float(theta if theta is not None else known if known is not None else 10000.0)
    kind = sc.get("rope_type", sc.get("type", "default"))
    if kind not in _KIND_KEYS:
        raise ValueError(f"rotary_tables: unknown rope_type {kind!r}")
    unread = sorted(str(k) for k, v in sc.items() if v is not None and k not in _KEYS | _KIND_KEYS[kind])
    if unread:
        raise ValueError(f"rotary_tables: rope_type {kind!r} does not read {', '.join(unread)}")
    f64 = dict(dtype=torch.float64, device=device)
    trained = sc.get("original_max_position_embeddings") or sc.get("max_position_embeddings")
    if kind == "dynamic":                                   # (what such a model counts from is its maximum)
        trained = sc.get("max_position_embeddings") or trained
    if kind in ("dynamic", "yarn", "llama3", "longrope") and not trained:
        raise ValueError(f"rotary_tables: rope_type {kind!r} needs original_max_position_embeddings")
    if kind in ("linear", "dynamic", "yarn", "llama3") and not sc.get("factor", 0) >= 1:
        raise ValueError(f"rotary_tables: rope_type {kind!r} needs a factor of at least 1")
    factor, amp = float(sc.get("factor") or 1.0), 1.0
    if kind == "dynamic" and length > trained:
        if part == 2:
            raise ValueError("rotary_tables: one pair has no slower one to stretch")
        theta = theta * (factor * length / trained - (factor - 1)) ** (part / (part - 2))
    inv = theta ** (-torch.arange(0, part, 2, **f64) / part)
    if kind == "linear":
        inv = inv / factor
    elif kind == "yarn":
        pair = lambda turns: part * math.log(trained / (turns * 2 * math.pi)) / (2 * math.log(theta))        # noqa: E731
        lo, hi = pair(float(sc.get("beta_fast") or 32.0)), pair(float(sc.get("beta_slow") or 1.0))
        if sc.get("truncate", True):
            lo, hi = math.floor(lo), math.ceil(hi)
        lo, hi = max(0, lo), min(part - 1, hi)
        slow = ((torch.arange(part // 2, **f64) - lo) / max(hi - lo, 1e-3)).clamp(0, 1)
        inv = inv * (1 - slow) + inv / factor * slow
        given, m, a = sc.get("attention_factor"), sc.get("mscale"), sc.get("mscale_all_dim")
        grown = lambda by: 0.1 * float(by) * math.log(factor) + 1.0                                          # noqa: E731
        amp = float(given) if given is not None else grown(m) / grown(a) if m and a else grown(1.0)
    elif kind == "llama3":
        low, high = float(sc.get("low_freq_factor", 1.0)), float(sc.get("high_freq_factor", 4.0))
        turns = trained * inv / (2 * math.pi)
        keep = ((turns - low) / max(high - low, 1e-12)).clamp(0, 1)
        inv = inv * keep + inv / factor * (1 - keep)
    elif kind == "longrope":
        by = sc.get("long_factor" if length > trained else "short_factor")
        if by is None or len(by) != part // 2:
            raise ValueError(f"rotary_tables: longrope needs {part // 2} factors")
        inv = inv / torch.tensor(by, **f64)
        given, stretch = sc.get("attention_factor"), sc.get("factor")
        if stretch is None and sc.get("max_position_embeddings"):
            stretch = sc["max_position_embeddings"] / trained
        if given is None and stretch is None:
            raise ValueError("rotary_tables: longrope needs factor, attention_factor or max_position_embeddings")
        amp = float(given) if given is not None else (math.sqrt(1 + math.log(stretch) / math.log(trained)) if stretch > 1 else 1.0)
    cos, sin = torch.empty(2, length, part // 2, dtype=torch.float32, device=device)
    step = max(1, (1 << 24) // part)                        # (in parts: the angles take twice the tables' bytes)
    for at in range(0, length, step):
        angle = torch.arange(at, min(length, at + step), **f64)[:, None] * inv
        cos[at:at + step], sin[at:at + step] = angle.cos() * amp, angle.sin() * amp
    return cos, sin


class _Rotate(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, cos, sin, interleaved, offset, inverse):
        ctx.save_for_backward(positions, cos, sin)
        ctx.how = interleaved, offset, inverse
        return _apply(q, k, positions, cos, sin, interleaved, offset, inverse, None, None, 0.0, None)

    @staticmethod
    def backward(ctx, gq, gk):
        interleaved, offset, inverse = ctx.how
        gq, gk = (None if g is None else g if g.stride(2) == 1 else g.contiguous() for g in (gq, gk))
        gq, gk = _Rotate.apply(gq, gk, *ctx.saved_tensors, interleaved, offset, not inverse)
        return gq, gk, None, None, None, None, None, None


def _apply(q, k, positions, cos, sin, interleaved, offset, inverse, q_norm, k_norm, eps, out):
    host = calls() if out is None else None
    if host is not None:
        done = host[0].rotate(host[1], q, k, positions, cos, sin, interleaved, offset, inverse, q_norm, k_norm, eps)
        if done is not None:
            return done if k is not None else (done, None)
    make = lambda t: None if t is None else torch.empty(t.shape, dtype=t.dtype, device=t.device)              # noqa: E731
    q_out, k_out = (make(q), make(k)) if out is None else (out[0], out[1])
    ext().rotate(q, k, positions, cos, sin, interleaved, offset, inverse, q_norm, k_norm, eps, q_out, k_out)
    return q_out, k_out


def _has_tangent(*tensors):
    """is one of the tensors a dual one of forward-mode differentiation"""
    return any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors)


def rotate(q, k, positions, cos, sin, interleaved=True, offset=0, q_norm=None, k_norm=None, eps=1e-6, inverse=False, out=None):
    """(q, k) rotated by their tokens' positions: q [N, Hq, D] and k [N, Hk, D] (or None) BF16, FP16 or float32, heads and tokens at any
    stride (parts of a fused q/k/v row); positions int64 [N] (or [1]: one for all; beyond the table: its last row); cos, sin float32
    [P, R / 2], R <= D.  The R values of every head from `offset` on are rotated, as pairs (2i, 2i + 1) or, with interleaved=False, (i, i +
    R / 2); the others pass through.  With q_norm / k_norm ([D], the values' type) heads are RMS-normalised before, all of their values.
    fp32 arithmetic, rounded once.  out: (q, k) outputs; an output may be its input.  inverse: by the opposite angles, so that it undoes
    a rotation (by tables without an amplitude).

    Gradients flow to q and k (not to tables or through norms, and not with `out`, which are refused; nor are there forward-mode derivatives: dual
    tensors are refused); they are the inverse rotation.  As for every function: before backward() is captured into a CUDA graph, let go of eager graphs over the same leaves."""
    # (a level of forward mode is open; where torch does not say so, it is looked for in the tensors)
    if getattr(forward_ad, "_current_level", 0) >= 0 and _has_tangent(q, k, cos, sin, q_norm, k_norm, *(out or ())):
        raise RuntimeError("rotate: no forward-mode derivatives")
    if torch.is_grad_enabled() and (q.requires_grad or cos.requires_grad or sin.requires_grad or (k is not None and k.requires_grad)
                                    or (q_norm is not None and q_norm.requires_grad) or (k_norm is not None and k_norm.requires_grad)
                                    or (out is not None and any(t is not None and t.requires_grad for t in out))):
        if q_norm is not None or k_norm is not None or out is not None or cos.requires_grad or sin.requires_grad:
            raise RuntimeError("rotate: gradients flow through the rotation of q and k alone (not to tables, norms and given outputs)")
        host = calls() if k is not None else None
        if host is not None:                                # (the same function in native code)
            done = host[0].rotate_grad(host[1], q, k, positions, cos, sin, interleaved, offset, inverse)
            if done is not None:
                return done
        if k is None:
            return _Rotate.apply(q, q[:, :0], positions, cos, sin, interleaved, offset, inverse)[0], None
        return _Rotate.apply(q, k, positions, cos, sin, interleaved, offset, inverse)
    return _apply(q, k, positions, cos, sin, interleaved, offset, inverse, q_norm, k_norm, eps, out)
