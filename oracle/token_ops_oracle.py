"""64-bit statements of the token-sequence operators (per-head norm with rotation, masked attention) and, with every result, the
largest error that 32-bit sums and the stated roundings to 16 bits allow, element by element.

Rounding counts used below, u = finfo(dtype).eps / 2 (relative half step of the 16-bit type):
  attention forward:  probabilities rounded once (relative u) before the product with v, the output once:
      |do| <= (u + SLACK) sum_j p_j |v_j| + u |o|;  f16 also loses up to 2^-25 absolute per probability (taken relative to a
      maximum, the sum is >= 1):  + 2^-25 sum_j |v_j|.
  SLACK covers the 32-bit arithmetic of scores, exponentials and sums: a score of size s in base 2 has an error of about
      (sqrt(D) + 4) 2^-24 |s|, a relative error ln 2 times that of the probability: below 1e-4 for |s| <= 150, D <= 128.
  Numbers below 2^-126 do not exist in 32 bits (nor in bf16): a probability or product under 1.2e-38 is lost, and the sums of
      up to 1e5 of them with operands under 100 stay below UNDER = 1e-30, which is added to every tolerance.
  backward: P and dS are rounded once each; delta is the row sum of do times the ROUNDED output, hence off by sum_d |do_d| tol(o_d).
"""
import math

import torch

SLACK = 1e-4
UNDER = 1e-30


def turned(x, cos, sin, interleaved):
    """x [..., R] with its pairs turned."""
    R = x.shape[-1]
    y = torch.empty_like(x)
    first, second = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
    a, b = x[..., first], x[..., second]
    y[..., first], y[..., second] = a * cos - b * sin, a * sin + b * cos
    return y


def norm_rope(x, weight, positions, frequencies, eps, interleaved, grad=None):
    """x [B, N, H, D] -> y (and dx, dw for `grad`), each with its tolerance: {"y": (value, tol), ...}."""
    u = torch.finfo(x.dtype).eps / 2 if x.dtype != torch.float32 else 2.0 ** -24
    R = 2 * frequencies.numel()
    xd = x.double()
    w = weight.double() if weight is not None else torch.ones(x.shape[-1], dtype=torch.float64, device=x.device)
    angle = (positions.double()[..., None] * frequencies).expand(x.shape[0], x.shape[1], R // 2)[:, :, None]
    cos, sin = angle.cos(), angle.sin()
    r = 1 / (xd.pow(2).mean(-1, keepdim=True) + eps).sqrt()
    n = xd * r

    def turn(t, s, absolute=False):
        c, d = (cos.abs(), -sin.abs()) if absolute else (cos, s * sin)
        a = turned(t[..., :R], c, d, interleaved)
        return torch.cat((a, t[..., R:]), -1)

    def mass(t):                       # |a| + |b| of every pair, |t| outside
        m = t.abs().clone()
        a = turned(m[..., :R], torch.ones_like(cos), torch.ones_like(cos), interleaved)      # (a - b, a + b)
        top = a.clone()
        first, second = (slice(0, R, 2), slice(1, R, 2)) if interleaved else (slice(0, R // 2), slice(R // 2, R))
        top[..., first] = a[..., second]
        m[..., :R] = top
        return m

    y = turn(n * w, 1)
    out = {"y": (y, u * y.abs() + 2e-6 * mass(n * w) + 2.0 ** -25)}
    if grad is not None:
        g = turn(grad.double(), -1)
        h = g * w
        dx = r * (h - n * (h * n).mean(-1, keepdim=True))
        size = r * (mass(grad.double()) * w.abs() + n.abs() * (mass(grad.double()) * (w * n).abs()).mean(-1, keepdim=True))
        out["dx"] = (dx, u * dx.abs() + 4e-6 * size + 2.0 ** -25)
        # 32-bit sums: at most a few hundred terms in a row per lane, then trees
        out["dw"] = ((g * n).sum((0, 1, 2)), 3e-5 * (mass(grad.double()) * n.abs()).sum((0, 1, 2)) + 1e-12)
    return out


def visible(B, Nq, Nk, device, causal=False, prefix=None, documents=None, lengths=None, starts=None):
    """(see [B, Nq, Nk], p [B, Nq])"""
    p = torch.arange(Nq, device=device)[None] + (starts.long()[:, None] if starts is not None else torch.full((B, 1), Nk - Nq, device=device))
    j = torch.arange(Nk, device=device)
    see = torch.ones(B, Nq, Nk, dtype=torch.bool, device=device)
    if causal:
        see = j[None, None] <= p[:, :, None]
        if prefix is not None:
            see = see | (j[None, None] < prefix.long()[:, None, None])
    if lengths is not None:
        see = see & (j[None, None] < lengths.long()[:, None, None])
    if documents is not None:
        inside = (p >= 0) & (p < Nk)
        mine = torch.where(inside, documents.long().gather(1, p.clamp(0, max(Nk - 1, 0))), torch.full_like(p, -1))
        see = see & (mine[:, :, None] == documents.long()[:, None]) & (mine[:, :, None] >= 0)
    return see, p


def attention(q, k, v, *, scale=None, softcap=None, slopes=None, causal=False, prefix=None, documents=None, lengths=None, starts=None,
              grad=None):
    """{"o": (value, tol)} and, with `grad`, dq, dk, dv.  Values at places that no row sees count as zeros."""
    B, Nq, Hq, D = q.shape
    Nk, Hk = k.shape[1:3]
    G, dt, dev = Hq // Hk, q.dtype, q.device
    u = torch.finfo(dt).eps / 2 if dt in (torch.bfloat16, torch.float16) else 0.0
    tiny = 2.0 ** -25 if dt == torch.float16 else UNDER
    scale = D ** -0.5 if scale is None else scale
    see, p = visible(B, Nq, Nk, dev, causal, prefix, documents, lengths, starts)
    used_k = see.any(1)[:, :, None, None]
    used_q = see.any(2)[:, :, None, None]
    Q = torch.where(used_q, q.double(), 0.0).transpose(1, 2)
    K = torch.where(used_k, k.double(), 0.0).transpose(1, 2).repeat_interleave(G, 1)
    V = torch.where(used_k, v.double(), 0.0).transpose(1, 2).repeat_interleave(G, 1)
    t = Q @ K.transpose(2, 3).contiguous() * scale
    cap = None
    if softcap:
        cap = torch.tanh(t / softcap)
        t = cap * softcap
    if slopes is not None:
        dist = (p[:, :, None] - torch.arange(Nk, device=dev)).abs().double()
        t = t - slopes.double()[None, :, None, None] * dist[:, None]
    t = t.masked_fill(~see[:, None], -math.inf)
    m = t.amax(-1, keepdim=True).clamp_min(-1e300) if Nk else torch.zeros(B, Hq, Nq, 1, dtype=torch.float64, device=dev)
    P = (t - m).exp()
    P = P / P.sum(-1, keepdim=True).clamp_min(1e-300)
    o = P @ V
    seen = see[:, None].double()
    tol = (u + SLACK) * (P @ V.abs()) + u * o.abs() + tiny * (1 + seen @ V.abs())
    back = lambda x: x.transpose(1, 2)                                          # noqa: E731
    out = {"o": (back(o), back(tol))}
    if grad is None:
        return out
    dO = torch.where(used_q, grad.double(), 0.0).transpose(1, 2)
    dP = dO @ V.transpose(2, 3).contiguous()
    delta = (dO * o).sum(-1, keepdim=True)
    dS = P * (dP - delta)
    size = dO.abs() @ V.abs().transpose(2, 3).contiguous() + (dO * o).abs().sum(-1, keepdim=True)     # what 32-bit sums of dP - delta run over
    ddelta = (dO.abs() * tol).sum(-1, keepdim=True)
    if cap is not None:
        dS = dS * (1 - cap * cap)
    err = (u + SLACK) * dS.abs() + P * (ddelta + SLACK * size * 0.1)
    shift = lambda a: tiny * a / 8                                              # noqa: E731  f16: absolute step of the scaled dS
    amax_i = dO.abs().amax(-1, keepdim=True)
    amax_g = dO.reshape(B, Hk, G * Nq * D).abs().amax(-1)[:, :, None, None].repeat_interleave(G, 1)
    fold = lambda x: back(x.reshape(B, Hk, G, Nk, D).sum(2))                    # noqa: E731
    dq = dS @ K * scale
    tq = ((err + shift(amax_i) * seen) @ K.abs()) * scale + u * dq.abs() + tiny
    St = dS.transpose(2, 3).contiguous()
    dk, dv = fold(St @ Q) * scale, fold(P.transpose(2, 3).contiguous() @ dO)
    tk = fold((err + shift(amax_g) * seen).transpose(2, 3).contiguous() @ Q.abs()) * scale + u * dk.abs() + tiny
    tv = fold(((u + SLACK) * P + tiny / 1024 * seen).transpose(2, 3).contiguous() @ dO.abs()) + u * dv.abs() + tiny
    out.update(dq=(back(dq), back(tq)), dk=(dk, tk), dv=(dv, tv))
    return out
