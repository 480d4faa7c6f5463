"""Token-sequence operators on the GPU (audio_diffusion_amd.transformer) against their 64-bit statements in
oracle/token_ops_oracle.py.  The tolerances come from that file: every element has its own, counted from the roundings that the
kernels make (see its docstring), and none of them was set after a run."""
import pytest
import torch

from oracle import token_ops_oracle as O

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def A():
    import audio_diffusion_amd as A
    assert torch.cuda.is_available(), "GPU tests need a ROCm device"
    return A


def gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def randn(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g, device="cuda") * scale).to(dtype)


def within(name, got, want):
    value, tol = want
    got = got.double()
    assert got.shape == value.shape, (name, got.shape, value.shape)
    bad = ~((got - value).abs() <= tol)
    if bool(bad.any()):
        at = tuple(int(x) for x in bad.nonzero()[0])
        raise AssertionError(f"{name}: {int(bad.sum())} of {bad.numel()} off, first at {at}: {float(got[at])} not {float(value[at])} +- {float(tol[at])}")


# ---- per-head norm and rotation -------------------------------------------------------------------------------------------

NORM_CASES = [
    # B, N, Hq, Hk, D, R, interleaved, layout
    (1, 1, 1, 1, 2, 2, False, "plain"),
    (3, 1, 32, 8, 128, 128, False, "plain"),          # one new token of each sequence
    (2, 5, 3, 1, 128, 64, False, "packed"),
    (2, 37, 5, 5, 64, 64, True, "packed"),
    (1, 130, 2, 2, 96, 96, False, "plain"),           # lanes without a part of the row
    (2, 17, 4, 2, 32, 16, True, "swapped"),
    (1, 9, 3, 3, 80, 40, False, "plain"),             # rotated part not whole pieces: element by element
    (1, 9, 3, 3, 80, 42, True, "plain"),              # pairs that end inside a piece
    (2, 11, 2, 2, 66, 66, False, "plain"),            # odd sizes
    (1, 7, 2, 1, 256, 256, False, "plain"),
    (1, 7, 2, 1, 254, 2, True, "offset"),             # rows that are not 16-byte aligned
    (1, 33, 1, 4, 128, 0, False, "plain"),            # norm only
    (2, 2100, 6, 2, 64, 32, False, "plain"),          # whole tokens per wave, several tokens per wave backwards
]


def layout(x, how):
    """The same values in another memory order."""
    B, N, H, D = x.shape
    if how == "swapped":                               # [B, H, N, D] in memory
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if how == "packed":                                # a slice of a wider projection
        wide = torch.full((B, N, H * D + 64), 7.0, dtype=x.dtype, device=x.device)
        view = wide[..., 32:32 + H * D].view(B, N, H, D)
        view.copy_(x)
        return view
    if how == "offset":
        flat = torch.empty(x.numel() + 1, dtype=x.dtype, device=x.device)[1:].view(x.shape)
        flat.copy_(x)
        return flat
    return x


@pytest.mark.parametrize("dt", ["f32", "bf16", "f16"])
@pytest.mark.parametrize("case", NORM_CASES, ids=lambda c: "-".join(map(str, c)))
def test_qk_norm_rope(A, case, dt):
    B, N, Hq, Hk, D, R, inter, how = case
    g = gen(N * 131 + D)
    dtype = DT[dt]
    q, k = randn(g, B, N, Hq, D, dtype=dtype, scale=1.7), randn(g, B, N, Hk, D, dtype=dtype, scale=0.4)
    q[0, 0, 0] = 0                                     # a row of zeros stays zeros
    wq, wk = 1 + randn(g, D, scale=0.3), 1 + randn(g, D, scale=0.3)
    pos = torch.randint(-50, 200000, (B, N), generator=g, device="cuda")
    f = A.rope_frequencies(R, device="cuda")
    dq, dk = randn(g, B, N, Hq, D, dtype=dtype), randn(g, B, N, Hk, D, dtype=dtype)
    leaves = [layout(q, how).detach().requires_grad_(), layout(k, how).detach().requires_grad_(), wq.clone().requires_grad_(), wk.clone().requires_grad_()]
    assert leaves[0].stride() == layout(q, how).stride()
    yq, yk = A.qk_norm_rope(*leaves, pos, f, eps=1e-6, interleaved=inter)
    assert yq.is_contiguous() and yk.is_contiguous() and yq.dtype == dtype
    gr = torch.autograd.grad((yq, yk), leaves, (layout(dq, how), layout(dk, how)))
    for x, w, d, y, gx, gw in ((q, wq, dq, yq, gr[0], gr[2]), (k, wk, dk, yk, gr[1], gr[3])):
        want = O.norm_rope(x, w, pos, f, 1e-6, inter, grad=d)
        within("y", y, want["y"])
        within("dx", gx, want["dx"])
        within("dw", gw, want["dw"])


def test_qk_norm_rope_positions_weights_and_types(A):
    g = gen(5)
    q, k = randn(g, 2, 6, 2, 64, dtype=torch.bfloat16), randn(g, 2, 6, 1, 64, dtype=torch.bfloat16)
    f = A.rope_frequencies(64, device="cuda")
    pos = torch.arange(6, device="cuda")
    y = A.qk_norm_rope(q, k, None, None, pos, f)
    for other in (pos.int(), pos.expand(2, 6), pos.int().repeat(2, 1), pos.repeat_interleave(2)[::2]):
        z = A.qk_norm_rope(q, k, None, None, other, f)
        assert torch.equal(y[0], z[0]) and torch.equal(y[1], z[1])
    within("y", y[0], O.norm_rope(q, None, pos[None], f, 1e-6, False)["y"])
    # weights of another type get gradients of that type
    w = torch.ones(64, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    z = A.qk_norm_rope(q, k, w, w, pos, f)
    (gw,) = torch.autograd.grad(z[0].float().sum() + z[1].float().sum(), w)
    assert gw.dtype == torch.bfloat16 and torch.equal(z[0], y[0])
    # far positions keep their angle: 2^40 turns the first pair by 2^40 radians
    far = torch.full((6,), 1 << 40, device="cuda")
    z = A.qk_norm_rope(q.float(), k.float(), None, None, far, f)
    within("far", z[0], O.norm_rope(q.float(), None, far[None], f, 1e-6, False)["y"])
    # an infinity or NaN stays in its own row, and beside the rotated part in its own element's formula
    bad = q.clone()
    bad[0, 2, 1, 3], bad[1, 4, 0, 60] = float("inf"), float("nan")
    z = A.qk_norm_rope(bad, k, None, None, pos, f)
    rows = torch.ones(2, 6, 2, dtype=torch.bool, device="cuda")
    rows[0, 2, 1] = rows[1, 4, 0] = False
    assert torch.equal(z[0][rows], y[0][rows]) and not bool(torch.isfinite(z[0][~rows]).all())
    # no rows
    e = A.qk_norm_rope(q[:, :0], k[:, :0], None, None, pos[:0], f)
    assert e[0].shape == (2, 0, 2, 64) and e[1].shape == (2, 0, 1, 64)


# ---- attention ------------------------------------------------------------------------------------------------------------

def ids(g, B, N, mean):
    """Documents of about `mean` tokens in rising order, some padding at the end of sample 0."""
    d = torch.cumsum(torch.rand(B, N, generator=g, device="cuda") < 1.0 / mean, 1).int()
    if N > 8:
        d[0, N - N // 8:] = -1
    return d


def whole(g, low, high, B):
    return torch.randint(low, high, (B,), generator=g, device="cuda", dtype=torch.int32)


ATT_CASES = {
    # name: B, Nq, Nk, Hq, Hk, D, options
    "one key": (1, 1, 1, 1, 1, 64, {}),
    "one row": (2, 1, 300, 4, 2, 128, dict(causal=True)),
    "whole": (2, 200, 200, 2, 2, 64, {}),
    "whole 32": (1, 257, 257, 3, 3, 32, dict(slopes=True)),
    "whole 128": (1, 300, 300, 2, 1, 128, {}),
    "cross": (2, 70, 333, 4, 2, 64, dict(slopes=True)),
    "cross long": (1, 300, 65, 2, 2, 128, dict(causal=True)),               # rows before the first key see nothing
    "causal": (1, 513, 513, 2, 1, 128, dict(causal=True)),
    "causal cap": (2, 130, 130, 4, 1, 64, dict(causal=True, softcap=8.0)),
    "cap slopes": (1, 190, 190, 3, 3, 32, dict(softcap=15.0, slopes=True, causal=True)),
    "prefix": (3, 400, 400, 2, 2, 64, dict(causal=True, prefix=True)),
    "documents": (2, 515, 515, 2, 1, 128, dict(documents=90)),
    "documents causal": (2, 700, 700, 2, 2, 64, dict(documents=60, causal=True, softcap=20.0)),
    "documents short": (2, 600, 600, 4, 2, 32, dict(documents=3, causal=True)),
    "documents prefix": (2, 300, 300, 2, 2, 64, dict(documents=120, causal=True, prefix=True, slopes=True)),
    "lengths": (4, 150, 150, 2, 2, 128, dict(lengths=True)),
    "lengths causal": (4, 97, 290, 4, 4, 64, dict(lengths=True, causal=True, starts=True)),
    "lengths all": (3, 260, 260, 6, 2, 64, dict(lengths=True, causal=True, prefix=True, documents=80, softcap=10.0, slopes=True)),
    "step": (3, 1, 1100, 8, 2, 128, dict(lengths=True, causal=True, starts=True)),
    "step slopes": (5, 1, 700, 4, 4, 64, dict(lengths=True, causal=True, starts=True, slopes=True, softcap=30.0)),
    "step documents": (2, 1, 900, 6, 1, 32, dict(documents=200, causal=True)),
    "few rows": (2, 5, 2000, 16, 2, 128, dict(lengths=True, causal=True, starts=True)),
    "few rows many heads": (1, 7, 130, 40, 1, 64, dict(causal=True)),
    "long": (1, 2049, 2049, 4, 2, 64, dict(causal=True)),
}


def make(case, dtype, seed=0, scale=1.3):
    B, Nq, Nk, Hq, Hk, D, o = case
    g = gen(seed + Nq + 7 * Nk)
    q, k, v = (randn(g, *s, dtype=dtype, scale=scale) for s in ((B, Nq, Hq, D), (B, Nk, Hk, D), (B, Nk, Hk, D)))
    how = dict(causal=bool(o.get("causal")), softcap=o.get("softcap"))
    if o.get("slopes"):
        how["slopes"] = torch.exp2(-8.0 * torch.arange(1, Hq + 1, device="cuda") / Hq).float()
    if o.get("prefix"):
        how["prefix"] = whole(g, 0, Nk + 1, B)
    if o.get("documents"):
        how["documents"] = ids(g, B, Nk, o["documents"])
    if o.get("lengths"):
        how["lengths"] = whole(g, max(1, Nk // 3), Nk + 1, B)
        how["lengths"][0] = Nk
        if B > 2 and not o.get("starts"):
            how["lengths"][2] = 0                                              # a sample without keys
    if o.get("starts"):
        how["starts"] = (how["lengths"] - Nq).int()
    return q, k, v, randn(g, B, Nq, Hq, D, dtype=dtype), how


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("name", ATT_CASES)
def test_attention(A, name, dt):
    q, k, v, do, how = make(ATT_CASES[name], DT[dt])
    want = O.attention(q, k, v, grad=do, **how)
    o = A.masked_attention(q, k, v, **how)
    within("o", o, want["o"])
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o2 = A.masked_attention(*leaves, **how)
    within("o with gradients", o2, want["o"])
    for n, x in zip(("dq", "dk", "dv"), torch.autograd.grad(o2, leaves, do)):
        within(n, x, want[n])
