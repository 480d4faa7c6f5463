"""Cases of the token-sequence operators: ``qk_norm_rope`` (per-head RMS norm of queries and keys with the position
rotation) and ``masked_attention`` (scores capped by a tanh, biased by distance, under causal, prefix, document and length
masks), each forwards, with gradients, and for single tokens.

``run`` computes a case in its plain form, in elementary torch operations, or, with ``own`` set, by the package's operators.
``exact`` computes it in 64 bits.
"""
import math
import random  # noqa: F401  (draw() takes a random.Random)

import torch

own = False

TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BYTES = {"bf16": 2, "f16": 2, "f32": 4}
EPS = 1e-6


def rotate_case(name, type, B, N, Hq, Hk, D, R, train, interleaved=False, packed=False, far=0):
    return {"name": name, "op": "rotate", "type": type, "B": B, "N": N, "Hq": Hq, "Hk": Hk, "D": D, "R": R, "train": train,
            "interleaved": interleaved, "packed": packed, "far": far}


def attend_case(name, type, B, Nq, Nk, Hq, Hk, D, train=False, causal=False, prefix=False, documents=False, lengths=False,
                softcap=0.0, slopes=False):
    return {"name": name, "op": "attend", "type": type, "B": B, "Nq": Nq, "Nk": Nk, "Hq": Hq, "Hk": Hk, "D": D, "train": train,
            "causal": causal, "prefix": prefix, "documents": documents, "lengths": lengths, "softcap": softcap, "slopes": slopes}


def listed():
    return [
        # one new token of each of 32 sequences in generation, far into the sequence
        rotate_case("rotate_token", "bf16", 32, 1, 32, 8, 128, 128, False, far=100000),
        # a denoiser call over latent clips: views of one packed projection, half of each head rotated
        rotate_case("rotate_clips", "f16", 8, 4096, 16, 16, 64, 32, False, packed=True),
        # a training step over long token sequences of an odd length, shared key heads
        rotate_case("rotate_train", "bf16", 4, 8191, 32, 8, 128, 128, True),
        # a training step in full precision, adjacent pairs rotated
        rotate_case("rotate_train_f32", "f32", 2, 2049, 8, 8, 64, 64, True, interleaved=True),
        # one short clip at a deep level of the denoiser: 16 heads of 32, an odd length, distance bias
        attend_case("attend_short", "f16", 1, 257, 257, 16, 16, 32, slopes=True),
        # a batch of clips at a middle level: 8 heads of 64, distance bias in both directions
        attend_case("attend_clips", "bf16", 16, 1024, 1024, 8, 8, 64, slopes=True),
        # the prompt of a long generation: the prefix sees itself whole, the rest is causal, shared key heads
        attend_case("attend_prompt", "bf16", 2, 8192, 8192, 16, 4, 128, causal=True, prefix=True),
        # several documents in one row of an odd length, capped scores
        attend_case("attend_documents", "f16", 2, 4099, 4099, 16, 16, 64, documents=True, softcap=30.0),
        # one token over a short cache
        attend_case("step_short", "bf16", 4, 1, 1000, 8, 8, 64, causal=True, lengths=True),
        # one token over long caches of unequal fill, capped scores, shared key heads
        attend_case("step_long", "bf16", 8, 1, 65536, 32, 8, 128, causal=True, lengths=True, softcap=50.0),
        # a training step of a clip model: whole attention with distance bias
        attend_case("train_clips", "f16", 4, 4096, 4096, 16, 16, 64, train=True, slopes=True),
        # a training step over packed documents: causal, capped, shared key heads, an odd length
        attend_case("train_documents", "bf16", 1, 8190, 8190, 16, 4, 128, train=True, causal=True, documents=True, softcap=50.0),
    ]


def _spread(rng, low, high):
    """A whole number between low and high, even over its logarithm."""
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    if rng.random() < 0.35:
        while True:
            D = rng.choice((32, 64, 96, 128))
            Hk = rng.choice((1, 2, 4, 8, 16))
            c = rotate_case("", rng.choice(("bf16", "bf16", "f16", "f32")), _spread(rng, 1, 32), rng.choice((1, _spread(rng, 2, 8192))),
                            Hk * rng.choice((1, 1, 2, 4)), Hk, D, rng.choice((D, D // 2)), rng.random() < 0.5,
                            interleaved=rng.random() < 0.4, packed=rng.random() < 0.4, far=rng.choice((0, _spread(rng, 1, 1000000))))
            if c["B"] * c["N"] * (c["Hq"] + c["Hk"]) * D * BYTES[c["type"]] <= 4 * 8191 * 40 * 128 * 2:
                del c["name"]
                return c
    while True:
        D = rng.choice((32, 64, 64, 128, 128))
        Hk = rng.choice((1, 2, 4, 8, 16))
        Hq = Hk * rng.choice((1, 1, 2, 4))
        kind = rng.choice(("step", "whole", "train"))
        Nk = _spread(rng, 64, 65536 if kind == "step" else 8192)
        Nq = rng.choice((1, 1, rng.randint(1, 8))) if kind == "step" else rng.choice((Nk, Nk, _spread(rng, 1, Nk)))
        causal = kind == "step" or rng.random() < 0.5
        c = attend_case("", rng.choice(("bf16", "f16")), _spread(rng, 1, 16), Nq, Nk, Hq, Hk, D, train=kind == "train", causal=causal,
                        prefix=causal and kind != "step" and rng.random() < 0.3, documents=kind != "step" and rng.random() < 0.4,
                        lengths=kind == "step" or rng.random() < 0.3, softcap=rng.choice((0.0, 0.0, 20.0, 50.0)), slopes=rng.random() < 0.4)
        pairs, keys = c["B"] * Hq * Nq * Nk, c["B"] * Nk * Hk * D
        # no more scores and products than the largest whole case has, and no longer caches than the longest
        if pairs <= (16 * 8190 * 8190 if c["train"] else 2 * 16 * 8192 * 8192) and pairs * D <= (1 if c["train"] else 2) * 16 * 8190 * 8190 * 128 \
                and keys <= 8 * 65536 * 8 * 128:
            del c["name"]
            return c


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = TYPES[case["type"]]

    def normal(*shape, scale=1.0, dtype=dt):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)

    def whole(low, high, *shape):
        return torch.randint(low, high, shape, generator=g, device="cuda", dtype=torch.int32)

    B, Hq, Hk, D = case["B"], case["Hq"], case["Hk"], case["D"]
    s = {"case": case}
    if case["op"] == "rotate":
        N, R = case["N"], case["R"]
        if case["packed"]:                       # q, k and v of one projection: rows of [q | k | v]
            rows = normal(B, N, (Hq + 2 * Hk) * D, scale=1.5)
            s["q"] = rows[..., :Hq * D].view(B, N, Hq, D)
            s["k"] = rows[..., Hq * D:(Hq + Hk) * D].view(B, N, Hk, D)
        else:
            s["q"], s["k"] = normal(B, N, Hq, D, scale=1.5), normal(B, N, Hk, D, scale=1.5)
        s["q_weight"] = 1 + normal(D, scale=0.2, dtype=torch.float32)
        s["k_weight"] = 1 + normal(D, scale=0.2, dtype=torch.float32)
        s["positions"] = torch.arange(N, device="cuda")[None] + whole(case["far"] // 2, case["far"] + 1, B, 1)
        s["frequencies"] = 10000.0 ** (-torch.arange(R // 2, device="cuda", dtype=torch.float64) * 2 / R)
        if case["train"]:
            s["dq"], s["dk"] = normal(B, N, Hq, D), normal(B, N, Hk, D)
        return s
    Nq, Nk = case["Nq"], case["Nk"]
    # queries and keys as a norm over each head leaves them, with gains a little over one
    s["q"], s["k"], s["v"] = normal(B, Nq, Hq, D, scale=1.3), normal(B, Nk, Hk, D, scale=1.3), normal(B, Nk, Hk, D)
    s["lengths"] = s["starts"] = s["prefix"] = s["documents"] = s["slopes"] = None
    if case["lengths"]:
        s["lengths"] = whole(max(Nq, Nk // 2), Nk + 1, B) if Nk > Nq else whole(max(1, Nk // 2), Nk + 1, B)
        if Nq < Nk:                              # new tokens stand at the end of each sequence's filled part
            s["starts"] = (s["lengths"] - Nq).to(torch.int32)
    if case["prefix"]:
        s["prefix"] = whole(0, Nk // 2 + 1, B)
    if case["documents"]:                        # about five documents in a row, and some padding behind the last
        ends = torch.rand(B, Nk, generator=g, device="cuda") < 4.0 / Nk
        s["documents"] = torch.cumsum(ends, 1).to(torch.int32)
        s["documents"][:, Nk - Nk // 50:] = -1
    if case["slopes"]:
        s["slopes"] = torch.exp2(-8.0 * torch.arange(1, Hq + 1, device="cuda") / Hq).float()
    if case["train"]:
        s["do"] = normal(B, Nq, Hq, D)
    return s


def run(s):
    c = s["case"]
    if own:
        return _own_rotate(s, c) if c["op"] == "rotate" else _own_attend(s, c)
    return _plain_rotate(s, c) if c["op"] == "rotate" else _plain_attend(s, c)


# ---- the package's operators -------------------------------------------------------------------------------------------

def _own_rotate(s, c):
    from audio_diffusion_amd import qk_norm_rope
    if not c["train"]:
        return qk_norm_rope(s["q"], s["k"], s["q_weight"], s["k_weight"], s["positions"], s["frequencies"], eps=EPS,
                            interleaved=c["interleaved"])
    leaves = [s[n].detach().requires_grad_() for n in ("q", "k", "q_weight", "k_weight")]
    q, k = qk_norm_rope(*leaves, s["positions"], s["frequencies"], eps=EPS, interleaved=c["interleaved"])
    return (q.detach(), k.detach()) + torch.autograd.grad((q, k), leaves, (s["dq"], s["dk"]))


def _own_attend(s, c):
    from audio_diffusion_amd import masked_attention
    how = dict(softcap=c["softcap"] or None, slopes=s["slopes"], causal=c["causal"], prefix=s["prefix"], documents=s["documents"],
               lengths=s["lengths"], starts=s["starts"])
    if not c["train"]:
        return masked_attention(s["q"], s["k"], s["v"], **how)
    leaves = [s[n].detach().requires_grad_() for n in ("q", "k", "v")]
    o = masked_attention(*leaves, **how)
    return (o.detach(),) + torch.autograd.grad(o, leaves, s["do"])


# ---- the plain forms, in 32 bits ---------------------------------------------------------------------------------------

def _turned(x, cos, sin, R, interleaved):
    """The first R elements of each head turned by the angles, pair by pair."""
    a, b = (x[..., 0:R:2], x[..., 1:R:2]) if interleaved else (x[..., :R // 2], x[..., R // 2:R])
    u, v = a * cos - b * sin, a * sin + b * cos
    pair = torch.stack((u, v), -1).flatten(-2) if interleaved else torch.cat((u, v), -1)
    return torch.cat((pair, x[..., R:]), -1)


def _plain_rotate(s, c):
    R, inter = c["R"], c["interleaved"]
    angle = s["positions"].double()[..., None] * s["frequencies"]              # far positions need 64 bits
    cos, sin = angle.cos().float()[:, :, None], angle.sin().float()[:, :, None]
    qf, kf = s["q"].float(), s["k"].float()
    qr, kr = (torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) for x in (qf, kf))
    out = (_turned(qf * qr * s["q_weight"], cos, sin, R, inter).to(s["q"].dtype),
           _turned(kf * kr * s["k_weight"], cos, sin, R, inter).to(s["k"].dtype))
    if not c["train"]:
        return out
    gq, gk = _turned(s["dq"].float(), cos, -sin, R, inter), _turned(s["dk"].float(), cos, -sin, R, inter)
    hq, hk = qf * qr, kf * kr                                                  # the normalised rows
    wq, wk = (gq * hq).sum((0, 1, 2)), (gk * hk).sum((0, 1, 2))
    gq, gk = gq * s["q_weight"], gk * s["k_weight"]
    dq = qr * (gq - hq * (gq * hq).mean(-1, keepdim=True))
    dk = kr * (gk - hk * (gk * hk).mean(-1, keepdim=True))
    return out + (dq.to(s["q"].dtype), dk.to(s["k"].dtype), wq, wk)


def _visible(s, c, device):
    """[B, Nq, Nk]: which keys each query sees; and [B, Nq, 1], [1, 1, Nk]: their positions."""
    B, Nq, Nk = c["B"], c["Nq"], c["Nk"]
    start = s["starts"].long()[:, None] if s["starts"] is not None else torch.full((B, 1), Nk - Nq, device=device)
    i = (start + torch.arange(Nq, device=device))[:, :, None]
    j = torch.arange(Nk, device=device)[None, None, :]
    see = torch.ones(B, Nq, Nk, dtype=torch.bool, device=device)
    if c["causal"]:
        see &= (j <= i) if s["prefix"] is None else (j <= i) | (j < s["prefix"].long()[:, None, None])
    if s["lengths"] is not None:
        see &= j < s["lengths"].long()[:, None, None]
    if s["documents"] is not None:
        d = s["documents"].long()
        mine = torch.gather(d, 1, i[:, :, 0].clamp(0, Nk - 1))[:, :, None]
        see &= (mine == d[:, None, :]) & (mine >= 0) & (i >= 0) & (i < Nk)
    return see, i, j


def _plain_attend(s, c):
    B, Nq, Nk, Hq, Hk, D = (c[n] for n in ("B", "Nq", "Nk", "Hq", "Hk", "D"))
    G = Hq // Hk
    q = s["q"].float().view(B, Nq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Nq, D)
    k, v = (s[n].float().permute(0, 2, 1, 3).contiguous() for n in ("k", "v"))
    kt = k.transpose(2, 3).contiguous()
    see, i, j = _visible(s, c, q.device)
    see = see[:, None, None]
    t = (q @ kt).mul_(D ** -0.5).view(B, Hk, G, Nq, Nk)
    cap = None
    if c["softcap"]:
        cap = t.div_(c["softcap"]).tanh_()
        t = cap * c["softcap"]
    if c["slopes"]:
        t = t - s["slopes"].view(Hk, G, 1, 1) * (i - j).abs().float()[:, None, None]
    t = t.masked_fill_(~see, -math.inf)
    top = t.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, torch.zeros_like(top), top)            # a row that sees nothing
    p = t.sub_(top).exp_()
    p /= p.sum(-1, keepdim=True).clamp_min(1e-30)
    o = (p.view(B, Hk, G * Nq, Nk) @ v).view(B, Hk, G, Nq, D)

    def back(x):
        return x.permute(0, 3, 1, 2, 4).reshape(B, Nq, Hq, D).to(s["q"].dtype)

    if not c["train"]:
        return back(o)
    do = s["do"].float().view(B, Nq, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hk, G * Nq, D)
    dv = p.view(B, Hk, G * Nq, Nk).transpose(2, 3) @ do
    ds = (do @ v.transpose(2, 3).contiguous()).view(B, Hk, G, Nq, Nk)
    ds -= (p * ds).sum(-1, keepdim=True)
    ds *= p
    if cap is not None:
        ds *= 1 - cap * cap
    ds = ds.mul_(D ** -0.5).view(B, Hk, G * Nq, Nk)
    dq, dk = ds @ k, ds.transpose(2, 3) @ q
    return back(o), back(dq.view(B, Hk, G, Nq, D)), dk.transpose(1, 2).to(s["k"].dtype), dv.transpose(1, 2).to(s["v"].dtype)


# ---- in 64 bits, from the definitions ----------------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return _exact_rotate(s, case) if case["op"] == "rotate" else _exact_attend(s, case)


def _exact_rotate(s, c):
    R, outs, grads = c["R"], [], []
    turn = torch.polar(torch.ones_like(s["positions"][..., None] * s["frequencies"]), s["positions"][..., None] * s["frequencies"])
    for n in ("q", "k"):
        x, w = s[n].double().requires_grad_(c["train"]), s[n + "_weight"].double().requires_grad_(c["train"])
        y = x / (x.pow(2).sum(-1, keepdim=True) / c["D"] + EPS).sqrt() * w
        pairs = y[..., :R].unflatten(-1, (R // 2, 2) if c["interleaved"] else (2, R // 2))
        pairs = pairs if c["interleaved"] else pairs.transpose(-1, -2)
        z = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, :, None])
        z = (z if c["interleaved"] else z.transpose(-1, -2)).flatten(-2)
        y = torch.cat((z, y[..., R:]), -1)
        outs.append(y.detach())
        if c["train"]:
            grads.append(torch.autograd.grad(y, (x, w), s["d" + n].double()))
    if not c["train"]:
        return tuple(outs)
    return outs[0], outs[1], grads[0][0], grads[1][0], grads[0][1], grads[1][1]


def _exact_attend(s, c):
    Nq, Nk, G, D = c["Nq"], c["Nk"], c["Hq"] // c["Hk"], c["D"]
    q, k, v = (s[n].double() for n in ("q", "k", "v"))
    out, dq, dk, dv = torch.zeros_like(q), torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
    j = torch.arange(Nk, device=q.device)
    for b in range(c["B"]):
        i = torch.arange(Nq, device=q.device) + (int(s["starts"][b]) if s["starts"] is not None else Nk - Nq)
        hidden = torch.zeros(Nq, Nk, dtype=torch.bool, device=q.device)
        if c["causal"]:
            hidden |= j[None] > i[:, None]
            if s["prefix"] is not None:
                hidden &= (j >= int(s["prefix"][b]))[None]
        if s["lengths"] is not None:
            hidden |= (j >= int(s["lengths"][b]))[None]
        if s["documents"] is not None:
            d = s["documents"][b]
            own_id = torch.where((i >= 0) & (i < Nk), d[i.clamp(0, Nk - 1)], torch.full_like(i, -1).int())
            hidden |= (own_id[:, None] != d[None]) | (own_id < 0)[:, None]
        empty = hidden.all(1)
        for h in range(c["Hq"]):
            x, y, z = (t.detach().clone().requires_grad_(c["train"]) for t in (q[b, :, h], k[b, :, h // G], v[b, :, h // G]))
            t = x @ y.T / math.sqrt(D)
            if c["softcap"]:
                t = torch.tanh(t / c["softcap"]) * c["softcap"]
            if c["slopes"]:
                t = t - s["slopes"][h].double() * (i[:, None] - j[None]).abs()
            t = t.masked_fill(hidden, -math.inf).masked_fill(empty[:, None], 0.0)
            o = (torch.softmax(t, -1) @ z).masked_fill(empty[:, None], 0.0)
            out[b, :, h] = o.detach()
            if c["train"]:
                a, e, f = torch.autograd.grad(o, (x, y, z), s["do"][b, :, h].double())
                dq[b, :, h] = a
                dk[b, :, h // G] += e
                dv[b, :, h // G] += f
    return (out, dq, dk, dv) if c["train"] else out


# ---- what a case cannot do without -------------------------------------------------------------------------------------

def _pairs(c):
    """Query-key pairs of one head that a case has to look at: half for a causal one, a fifth for five documents."""
    Nq, Nk = c["Nq"], c["Nk"]
    n = Nq * Nk
    if c["causal"]:
        n -= Nq * (Nq - 1) / 2
        if c["prefix"]:                          # a prefix of a quarter of the row sees itself whole
            n += min(Nq, Nk / 4) ** 2 / 2
    if c["documents"]:
        n *= 0.33                                # documents of uneven lengths: the mean of their squared shares
    if c["lengths"]:
        n *= 0.75
    return c["B"] * n


def work(case):
    c, w = case, BYTES[case["type"]]
    if c["op"] == "rotate":
        n = c["B"] * c["N"] * (c["Hq"] + c["Hk"]) * c["D"]
        # forwards: read and write every element; with gradients: also read it and its gradient again and write one
        return {"bytes": float(n * w * (5 if c["train"] else 2)), "flops": float(n * (20 if c["train"] else 8))}
    filled = 0.75 if c["lengths"] else 1.0
    qb, kb = c["B"] * c["Nq"] * c["Hq"] * c["D"] * w, c["B"] * c["Nk"] * c["Hk"] * c["D"] * w
    flops = 4.0 * _pairs(c) * c["Hq"] * c["D"]
    if not c["train"]:
        return {"bytes": 2.0 * qb + 2.0 * kb * filled, "flops": flops}
    # q, k, v, o, do read; o, dq, dk, dv written; five products more or less the size of the two forwards
    return {"bytes": 5.0 * qb + 4.0 * kb, "flops": 3.5 * flops}
