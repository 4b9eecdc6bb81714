"""CPU oracle of the 4-bit key/value cache (test infrastructure only): the
quantiser, the byte layout and the attention, from their definitions in
include/llmx_attn.h, one token and one sequence at a time where that is the
plainest."""

from __future__ import annotations

import math
from typing import Optional

import torch

GROUP = 64


def quantise(x: torch.Tensor):
    """(codes int64 [..., D], s, m [..., D / 64] in x's dtype) of x [..., D]."""
    y = x.reshape(*x.shape[:-1], x.shape[-1] // GROUP, GROUP)
    m = y.amin(-1)
    # fp64 holds the difference and the quotient well enough that rounding
    # them to fp32 is what fp32 arithmetic gives.
    r = ((y.amax(-1).double() - m.double()).float().double() / 15.0).float()
    s = r.to(x.dtype)
    bumped = (s.view(torch.int16) + 1).view(x.dtype)
    s = torch.where(s.float() < r, bumped, s)
    # At the end of the type: the next s below where 15 s + m would round to infinity.
    past = (15.0 * s.double() + m.double()).float().to(x.dtype).isinf() & r.isfinite()
    s = torch.where(past, (s.view(torch.int16) - 1).view(x.dtype), s)
    s = torch.where(r.isfinite(), s, torch.full_like(s, float("nan")))
    diff = (y.double() - m.double()[..., None]).float().double()
    q = (diff / s.double()[..., None]).float()
    n = torch.where(s.float()[..., None] > 0, q, torch.zeros_like(q)).nan_to_num(0.0).round().clamp(0, 15)
    return n.reshape(x.shape).long(), s, m


def spread(p: torch.Tensor) -> torch.Tensor:
    """Per-group parameters [..., G] to channels [..., 64 G], in fp64."""
    return p.double().repeat_interleave(GROUP, -1)


def values(x: torch.Tensor):
    """What the cache holds for x: (n s + m in fp64, the read-back in x's dtype)."""
    n, s, m = quantise(x)
    v = n.double() * spread(s) + spread(m)
    back = (n.float() * spread(s).float() + spread(m).float()).to(x.dtype)  # n s is exact in fp32
    return v, back


def tile_bytes(head_dim: int) -> int:
    return 18 * head_dim


def word_offsets(head_dim: int, tok: int, chunk: int, is_v: bool) -> int:
    """Byte offset in a tile of the word of channels [8 chunk, 8 chunk + 8) of token tok."""
    G = head_dim // GROUP
    h = chunk // 8
    if not is_v:
        t, w = (chunk % 8) // 2, chunk % 2
        r, g = tok // 8, tok % 8
        x, base = (r * G + h) * 2 + w, 0
    else:
        g = chunk % 8
        a, t, c = tok // 8, (tok % 8) // 2, tok % 2
        x, base = (2 * a + c) * G + h, 8 * head_dim
    return base + (x // 4) * 512 + (4 * g + t) * 16 + (x % 4) * 4


def param_offset(head_dim: int, tok: int, is_v: bool, h: int) -> int:
    G = head_dim // GROUP
    return 16 * head_dim + ((tok * 2 + int(is_v)) * G + h) * 4


def write_token(tile: torch.Tensor, tok: int, k: torch.Tensor, v: torch.Tensor) -> None:
    """Writes token tok of a tile (uint8 [18 D]) from k, v [D]."""
    D = k.shape[-1]
    for is_v, x in ((False, k), (True, v)):
        n, s, m = quantise(x)
        for chunk in range(D // 8):
            at = word_offsets(D, tok, chunk, is_v)
            for i in range(4):
                tile[at + i] = int(n[8 * chunk + 2 * i]) | (int(n[8 * chunk + 2 * i + 1]) << 4)
        for h in range(D // GROUP):
            at = param_offset(D, tok, is_v, h)
            tile[at:at + 4] = torch.stack([s[h], m[h]]).view(torch.uint8)


def attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, q_len: int, kv_len: int, *, sm_scale: float,
              causal: bool = True, window: int = -1, cap: float = 0.0, slopes: Optional[torch.Tensor] = None):
    """One sequence in fp64: q [S, H, D] and the cached x = raw keys / values
    [N, Hkv, D] (quantised here).  Returns (o, lse, bound, lse_bound): the output, the
    log-sum-exp, how far a kernel that keeps its sums in fp32 and rounds q to 16
    bits of its row's maximum and p s to fp16 may be from the output, before the
    output's own rounding, and how far from the log-sum-exp."""
    S, H, D = q.shape
    Hkv = k.shape[1]
    o = torch.zeros(S, H, D, dtype=torch.float64)
    lse = torch.full((H, S), -math.inf, dtype=torch.float64)
    bound = torch.zeros_like(o)
    lse_bound = torch.zeros_like(lse)
    if kv_len == 0 or q_len == 0:
        return o, lse, bound, lse_bound
    k, v = k[:kv_len], v[:kv_len]
    kn, ks, km = quantise(k)
    kd = kn.double() * spread(ks) + spread(km)
    ka = kn.double() * spread(ks) + spread(km).abs()
    vn, vs, vm = quantise(v)
    vc = (vn.double() - 8) * spread(vs)
    va = spread(vm) + 8 * spread(vs)
    j = torch.arange(kv_len)
    i = torch.arange(q_len)[:, None]
    diag = i + kv_len - q_len
    seen = torch.ones(q_len, kv_len, dtype=torch.bool)
    if causal:
        seen &= j <= diag
    if window >= 0:
        seen &= diag - j <= window
    for h in range(H):
        g = h // (H // Hkv)
        s = q[:q_len, h].double() @ kd[:, g].T * sm_scale
        mag = q[:q_len, h].double().abs() @ ka[:, g].T * abs(sm_scale)
        # fp32 sums of at most 64 terms of size <= mag a group (2^-17 mag), and
        # a handful of fp32 roundings of the score itself.
        off = mag * 2.0 ** -17 + s.abs() * 2.0 ** -21
        # q as an integer of at most 32512: half a step (and fp32's rounding of the product) a channel, which
        # meets n - 8, and half a step a group from the rounding of what corrects for the 8.
        step = q[:q_len, h].double().abs().amax(-1, keepdim=True) / 32512
        off = off + step * (0.51 * ((kn[:, g].double() - 8).abs() * spread(ks)[:, g]).sum(-1)
                            + 0.51 * ks[:, g].double().sum(-1)) * abs(sm_scale)
        if cap > 0:
            s = cap * torch.tanh(s / cap)
            off = off + cap * 2.0 ** -21  # tanhf: 2 ulp of at most 1
        if slopes is not None:
            bias = float(slopes[h].float()) * j.double()
            s = s + bias
            off = off + (bias.abs() + s.abs()) * 2.0 ** -21
        s = s.masked_fill(~seen, -math.inf)
        top = s.amax(-1, keepdim=True)
        none = top == -math.inf
        p = torch.exp(s - top.masked_fill(none, 0.0))
        l = p.sum(-1, keepdim=True)
        p = p / l.masked_fill(none, 1.0)
        lse[h, :q_len] = (top + torch.log(l))[:, 0]
        o[:q_len, h] = p @ (vc[:, g] + va[:, g])
        # A log-sum-exp moves by no more than the largest of its scores does; 2^-20 for the sum's terms
        # (N 2^-23 more) and the logarithm, 2^-20 of its size for the roundings of a biased one.
        worst = off.masked_fill(~seen, 0.0).amax(-1)
        lse_bound[h, :q_len] = worst + 2.0 ** -20 + kv_len * 2.0 ** -23 + lse[h, :q_len].abs().nan_to_num(0, 0, 0) * 2.0 ** -20
        # Relative error of p: the score's, the exponential's, the sums' (N terms).
        rho = torch.expm1(2 * off.masked_fill(~seen, 0.0).amax(-1, keepdim=True)) + 2.0 ** -20 + kv_len * 2.0 ** -23
        size = p @ (vc[:, g].abs() + va[:, g].abs())
        # p s in fp16: half an ulp (2^-11), or below fp16's normal range 2^-25
        # of a scale that puts the largest s (or 2^-20 of a centre) that the row sees at 2^7 at least.
        widest = torch.maximum(spread(vs)[:, g], (spread(vm) + 8 * spread(vs))[:, g].abs() * 2.0 ** -20)
        widest = widest.double().nan_to_num(0.0, 0.0, 0.0).amax(-1)  # [N]: of the token's groups
        tiny = kv_len * 8 * 2.0 ** -32 * torch.where(seen, widest, 0.0).amax(-1, keepdim=True)
        bound[:q_len, h] = p @ vc[:, g].abs() * 2.0 ** -11 + 2 * rho * size + tiny
    return o, lse, bound, lse_bound
