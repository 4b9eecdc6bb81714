"""Oracle of the attention over a paged 16-bit cache, of its key weights and of
eviction, in 64 bits, with bounds of what the kernels' roundings may cost.

Test infrastructure only."""
import math

import torch


def attention(q, k, v, q_len, kv_len, *, sm_scale, causal=True, window=-1, cap=0.0, slopes=None, cap_relative=False):
    """One sequence: q [S, H, D], k and v [N, H_kv, D] (rows behind the lengths
    are not looked at).  Returns out [S, H, D], lse [H, S], weights [H_kv, N]
    and a bound for each, `out` without the rounding to its own type.

    The bounds add up, for a softmax weight p of a score x: half a step of the
    type for p's rounding in the product with V (fp16: of 2^10 p, half of its
    smallest number below the normal range), fp32 sums of the products (2^-24 for
    each of the D terms and 2^-22 for each 16 tokens, whose sums the tensor core
    may cut instead of rounding), 2^-22 for the exponential, and 2^-23 of the
    numbers that the score is made of.  A soft-cap adds 2^-21 of the cap, or with
    cap_relative 2^-20 of the capped score."""
    S, H, D = q.shape
    N, Hkv = k.shape[0], k.shape[1]
    G = H // Hkv
    dt = q.dtype
    half = torch.finfo(dt).eps / 2
    out = torch.zeros(S, H, D, dtype=torch.float64)
    lse = torch.full((H, S), -math.inf, dtype=torch.float64)
    weights = torch.zeros(Hkv, N, dtype=torch.float64)
    b_out, b_lse, b_w = torch.zeros_like(out), torch.zeros_like(lse), torch.zeros_like(weights)
    if q_len == 0 or kv_len == 0:
        return out, lse, weights, b_out, b_lse, b_w
    j = torch.arange(kv_len)
    diag = torch.arange(q_len)[:, None] + kv_len - q_len
    seen = torch.ones(q_len, kv_len, dtype=torch.bool)
    if causal:
        seen &= j <= diag
    if window >= 0:
        seen &= diag - j <= window
    any_seen = seen.any(-1)
    for h in range(H):
        kd, vd = k[:kv_len, h // G].double(), v[:kv_len, h // G].double()
        qd = q[:q_len, h].double()
        raw = qd @ kd.T * sm_scale
        mag = qd.abs() @ kd.abs().T * abs(sm_scale)
        x = torch.tanh(raw / cap) * cap if cap > 0 else raw
        slope = 0.0 if slopes is None else float(slopes[h].float())
        ref = torch.where(seen, j, -1).amax(-1) if slope >= 0 else torch.where(seen, j, kv_len).amin(-1)
        bias = slope * (j - ref[:, None]).double()
        x = (x + bias).masked_fill(~seen, -math.inf)
        top = x.amax(-1, keepdim=True).masked_fill(~any_seen[:, None], 0.0)
        e = torch.exp(x - top)
        total = e.sum(-1, keepdim=True)
        p = (e / total).nan_to_num(0.0)
        # Relative error of a weight before its rounding.
        d = (D + 8) * 2.0 ** -24 * mag + 2.0 ** -21 + 2.0 ** -22 * (mag + bias.abs() + top.abs())
        if cap > 0:
            d = d + (2.0 ** -20 * (torch.tanh(raw / cap) * cap).abs() if cap_relative else 2.0 ** -21 * cap)
        d = torch.where(p > 0, d, 0.0)
        sums = 2.0 ** -22 * (kv_len / 16 + 8)
        dsum = (p * d).sum(-1, keepdim=True) + sums
        tiny = 2.0 ** -34 * torch.where(seen, 1.0, 0.0).double() / total if dt == torch.float16 else torch.zeros_like(p)
        av = vd.abs()
        o = p @ vd
        ob = (p * (d + half + sums) + tiny) @ av + o.abs() * dsum
        out[:q_len, h] = torch.where(any_seen[:, None], o, 0.0)
        b_out[:q_len, h] = torch.where(any_seen[:, None], ob, 0.0)
        le = (top + total.log())[:, 0]
        shift = slope * ref.double()
        lse[h, :q_len] = torch.where(any_seen, le + shift, -math.inf)
        b_lse[h, :q_len] = dsum[:, 0] + 2.0 ** -22 * (1 + le.abs() + shift.abs())
        weights[h // G, :kv_len] += p.sum(0)
        b_w[h // G, :kv_len] += (p * (d + dsum + 2.0 ** -22 * (1 + top.abs()) + 2.0 ** -24 * q_len * G)).sum(0)
    return out, lse, weights, b_out, b_lse, b_w


def kept(weights, n, budget, recent, sinks):
    """Positions that eviction keeps of n tokens with these weights (a list or
    tensor of n numbers), ascending."""
    if n <= budget:
        return list(range(n))
    w = [-math.inf if math.isnan(x) else x for x in torch.as_tensor(weights)[:n].tolist()]
    mid = sorted(range(sinks, n - recent), key=lambda i: (-w[i], i))[:budget - sinks - recent]
    return list(range(sinks)) + sorted(mid) + list(range(n - recent, n))
