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
    # enough rows and heads for the kernel that splits only query rows (the ones above split the keys as well)
    "many whole": (8, 150, 150, 32, 8, 64, {}),
    "many whole 32": (6, 257, 257, 32, 32, 32, dict(slopes=True)),
    "many one tile": (16, 65, 40, 16, 4, 128, {}),
    "many two tiles": (16, 100, 128, 16, 16, 128, dict(causal=True, softcap=12.0)),
    "many causal": (4, 300, 300, 24, 8, 128, dict(causal=True)),
    "many cross": (6, 200, 65, 32, 32, 32, dict(causal=True)),
    "many long keys": (3, 129, 700, 64, 16, 64, dict(causal=True, slopes=True)),
    "many prefix": (4, 270, 270, 32, 4, 64, dict(causal=True, prefix=True, softcap=9.0)),
    "many documents": (4, 515, 515, 24, 6, 128, dict(documents=90)),
    "many short documents": (4, 600, 600, 16, 4, 64, dict(documents=4, causal=True)),
    "many padded": (5, 130, 130, 32, 8, 64, dict(documents=40, lengths=True)),
    "many lengths": (5, 131, 390, 32, 8, 128, dict(lengths=True, causal=True, starts=True)),
    "many all": (4, 260, 260, 24, 8, 128, dict(lengths=True, causal=True, prefix=True, documents=80, softcap=10.0, slopes=True)),
    "many all 64": (4, 260, 260, 32, 8, 64, dict(lengths=True, causal=True, prefix=True, documents=80, softcap=10.0, slopes=True)),
    "many all 32": (4, 260, 260, 32, 8, 32, dict(lengths=True, causal=True, prefix=True, documents=80, softcap=10.0, slopes=True)),
    "many long": (1, 2100, 2100, 16, 4, 128, dict(causal=True, documents=700)),
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


@pytest.mark.parametrize("dt", ["bf16", "f16"])
def test_attention_gradient_against_differences(A, dt):
    """<gradient, d> against a central difference of the 64-bit statement along a random direction d: the difference's own error is
    of order h^2 (third derivatives of the mean of a softmax are below 10 here), the gradient's is its tolerance."""
    for n, name in enumerate(("causal cap", "documents prefix", "lengths all")):
        q, k, v, do, how = make(ATT_CASES[name], DT[dt], seed=n)
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        grads = torch.autograd.grad(A.masked_attention(*leaves, **how), leaves, do)
        want = O.attention(q, k, v, grad=do, **how)
        g, h = gen(50 + n), 1e-4
        for t, gr, key in zip(range(3), grads, ("dq", "dk", "dv")):
            base = [q.double(), k.double(), v.double()]
            d = randn(g, *base[t].shape).double()
            ends = []
            for s in (h, -h):
                moved = list(base)
                moved[t] = base[t] + s * d
                ends.append(float((O.attention(*moved, **how)["o"][0] * do.double()).sum()))
            slope = (ends[0] - ends[1]) / (2 * h)
            got = float((gr.double() * d).sum())
            tol = float((want[key][1] * d.abs()).sum()) + 10 * h * h * float(do.double().abs().sum())
            assert abs(got - slope) <= tol, (name, key, got, slope, tol)


def poison(t, where, g):
    t = t.clone()
    bad = torch.tensor([float("inf"), float("-inf"), float("nan")], device="cuda", dtype=t.dtype)
    t[where] = bad[torch.randint(0, 3, t[where].shape, generator=g, device="cuda")]
    return t


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("case", [(1, 300, 300, 2, 1, 128, {}), (6, 300, 300, 16, 4, 128, {}), (2, 1500, 1500, 16, 16, 64, {}), (1, 4, 900, 8, 2, 64, {}), (1, 700, 700, 16, 8, 128, {}),
                                  (1, 1, 2500, 8, 1, 32, {})],
                         ids=lambda c: "-".join(map(str, c[:6])))
def test_attention_non_finite_values_in_hidden_places(A, case, dt):
    """Infinities and NaN reach exactly the rows and keys that see them."""
    B, Nq, Nk, Hq, Hk, D, _ = case
    q, k, v, do, how = make(case, DT[dt])
    g = gen(9)
    # keys that do not exist: nothing changes, bit for bit
    lengths = whole(g, Nk // 2, Nk - 3, B)
    beyond = torch.arange(Nk, device="cuda")[None] >= lengths[:, None]
    o = A.masked_attention(q, k, v, lengths=lengths)
    assert torch.equal(o, A.masked_attention(q, poison(k, beyond, g), poison(v, beyond, g), lengths=lengths))
    # padding and other documents
    docs = (torch.arange(Nk, device="cuda") * 5 // Nk).int().repeat(B, 1)
    docs[:, Nk - 2:] = -1
    bad = (docs == 1) | (docs < 0)
    start = torch.full((B,), Nk - Nq, device="cuda", dtype=torch.int32) if Nq < Nk else None
    for causal in (False, True):
        how = dict(documents=docs, causal=causal, starts=start)
        want = O.attention(q, k, v, grad=do, **how)
        rows = torch.gather(bad, 1, (torch.arange(Nq, device="cuda") + Nk - Nq).repeat(B, 1))           # of a poisoned document
        leaves = [t.requires_grad_() for t in (poison(q, rows, g), poison(k, bad, g), poison(v, bad, g))]
        o = A.masked_attention(*leaves, **how)
        grads = torch.autograd.grad(o, leaves, poison(do, rows, g))
        for n, x, clean in (("o", o, ~rows), ("dq", grads[0], ~rows), ("dk", grads[1], ~bad), ("dv", grads[2], ~bad)):
            within(n, x[clean], tuple(t[clean] for t in want[n]))
        assert not bool(grads[1][docs < 0].any()) and not bool(o[torch.gather(docs, 1, (torch.arange(Nq, device="cuda") + Nk - Nq).repeat(B, 1)) < 0].any())
    # a causal mask: one poisoned key in the last third, rows before it do not notice
    j = Nk - Nq + (2 * Nq) // 3
    at = torch.zeros(B, Nk, dtype=torch.bool, device="cuda")
    at[:, j] = True
    want = O.attention(q, k, v, causal=True)
    o = A.masked_attention(q, poison(k, at, g), poison(v, at, g), causal=True)
    before = (torch.arange(Nq, device="cuda") + Nk - Nq < j).repeat(B, 1)
    within("o", o[before], tuple(t[before] for t in want["o"]))
    assert not bool(torch.isfinite(o[~before]).all(-1).any())


SPLIT_CASES = {
    # few keys under many rows: the keys' gradients are summed in parts
    "heads": (1, 600, 130, 6, 2, 128, dict(causal=True)),
    "heads of one": (2, 520, 200, 8, 1, 64, dict(slopes=True)),
    "heads and rows": (1, 1400, 100, 4, 1, 128, {}),
    "rows": (2, 2100, 70, 1, 1, 32, dict(softcap=10.0)),
    "causal rows": (1, 2300, 2300, 2, 2, 64, dict(causal=True)),
    "documents": (1, 1500, 1500, 4, 1, 128, dict(documents=300, causal=True, softcap=12.0)),
    "all": (3, 1030, 1030, 6, 2, 64, dict(lengths=True, causal=True, prefix=True, documents=200, softcap=10.0, slopes=True)),
    "lengths": (3, 1100, 1210, 3, 1, 32, dict(lengths=True, causal=True, starts=True)),
}


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("name", SPLIT_CASES)
def test_attention_gradients_in_parts(A, name, dt):
    q, k, v, do, how = make(SPLIT_CASES[name], DT[dt], seed=3)
    want = O.attention(q, k, v, grad=do, **how)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = A.masked_attention(*leaves, **how)
    grads = torch.autograd.grad(o, leaves, do, retain_graph=True)
    for n, x in zip(("o", "dq", "dk", "dv"), (o,) + grads):
        within(n, x, want[n])
    assert all(torch.equal(x, y) for x, y in zip(grads, torch.autograd.grad(o, leaves, do)))


def test_attention_gradients_in_parts_keep_non_finite_values_to_what_sees_them(A):
    B, N, Hq, Hk, D = 1, 1400, 4, 1, 128
    q, k, v, do, _ = make((B, N, N, Hq, Hk, D, {}), torch.bfloat16, seed=4)
    docs = (torch.arange(N, device="cuda") * 3 // N).int()[None]
    bad = docs == 1
    want = O.attention(q, k, v, grad=do, documents=docs, causal=True)
    g = gen(10)
    leaves = [t.requires_grad_() for t in (poison(q, bad, g), poison(k, bad, g), poison(v, bad, g))]
    o = A.masked_attention(*leaves, documents=docs, causal=True)
    for n, x in zip(("o", "dq", "dk", "dv"), (o,) + torch.autograd.grad(o, leaves, poison(do, bad, g))):
        within(n, x[~bad], tuple(t[~bad] for t in want[n]))


KEY_SPLIT_CASES = {
    # few rows over many keys: the queries' gradients are summed in parts
    "whole": (1, 64, 2200, 4, 2, 128, {}),
    "one row": (2, 1, 3000, 2, 1, 64, dict(slopes=True)),
    "causal": (1, 300, 2300, 2, 2, 64, dict(causal=True, softcap=9.0)),
    "documents": (2, 70, 1500, 3, 1, 128, dict(documents=300, causal=True)),
    "lengths": (3, 40, 1300, 4, 2, 32, dict(lengths=True, causal=True, starts=True, slopes=True)),
    "all": (2, 1100, 1100, 2, 1, 128, dict(lengths=True, causal=True, prefix=True, documents=250, softcap=10.0, slopes=True)),
}


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("name", KEY_SPLIT_CASES)
def test_attention_query_gradients_in_parts(A, name, dt):
    q, k, v, do, how = make(KEY_SPLIT_CASES[name], DT[dt], seed=5)
    want = O.attention(q, k, v, grad=do, **how)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = A.masked_attention(*leaves, **how)
    grads = torch.autograd.grad(o, leaves, do, retain_graph=True)
    for n, x in zip(("o", "dq", "dk", "dv"), (o,) + grads):
        within(n, x, want[n])
    assert all(torch.equal(x, y) for x, y in zip(grads, torch.autograd.grad(o, leaves, do)))


def test_attention_extreme_mask_values(A):
    """The ends of int32 in prefix, lengths and starts are values like any other."""
    low, high = -2 ** 31, 2 ** 31 - 1
    q, k, v, do, _ = make((2, 70, 70, 2, 1, 64, {}), torch.bfloat16)
    i32 = lambda *x: torch.tensor(x, device="cuda", dtype=torch.int32)          # noqa: E731
    for how, same in (
        (dict(causal=True, prefix=i32(low, high)), dict(causal=True, prefix=i32(0, 70))),
        (dict(lengths=i32(low, high)), dict(lengths=i32(0, 70))),
        (dict(causal=True, starts=i32(low, high)), dict(causal=True, starts=i32(-70, 70))),
        (dict(causal=True, starts=i32(low, high), prefix=i32(5, low)), dict(causal=True, starts=i32(-70, 70), prefix=i32(5, 0))),
    ):
        got = []
        for h in (how, same):
            leaves = [t.detach().requires_grad_() for t in (q, k, v)]
            o = A.masked_attention(*leaves, **h)
            got.append((o.detach(),) + torch.autograd.grad(o, leaves, do) + (A.masked_attention(q[:, :1], k, v, **h),))
        assert all(torch.equal(x, y) for x, y in zip(*got)), how


def test_attention_layouts(A):
    """Views of one projection, other memory orders, unaligned and expanded tensors: the same bits as contiguous ones."""
    g = gen(3)
    B, N, Hq, Hk, D = 2, 150, 4, 2, 64
    rows = randn(g, B, N, (Hq + 2 * Hk) * D, dtype=torch.bfloat16)
    q, k, v = rows.view(B, N, Hq + 2 * Hk, D).split((Hq, Hk, Hk), 2)
    do = randn(g, B, N, Hq, D, dtype=torch.bfloat16)

    def run(q, k, v, do):
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = A.masked_attention(*leaves, causal=True, softcap=20.0)
        return (o,) + torch.autograd.grad(o, leaves, do)

    base = run(*(t.contiguous() for t in (q, k, v)), do)
    for how in ("plain", "swapped", "offset"):
        for x, y in zip(base, run(layout(q, how), layout(k, how), layout(v, how), layout(do, how))):
            assert torch.equal(x, y), how
    for x, y in zip(base, run(q, k, v, do.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0))):       # elements of a head apart
        assert torch.equal(x, y)
    # one sample's keys for all samples, one gradient for all heads
    one = k[:1].expand(B, N, Hk, D), v[:1].expand(B, N, Hk, D), do[:, :, :1].expand(B, N, Hq, D)
    for x, y in zip(run(q, *one), run(q, *(t.contiguous() for t in one))):
        assert torch.equal(x, y)
    # in reduced form the gradients of expanded leaves are summed
    kl = k[:1].contiguous().requires_grad_()
    o = A.masked_attention(q, kl.expand(B, N, Hk, D), v, causal=True)
    (dk,) = torch.autograd.grad(o, kl, do)
    assert dk.shape == kl.shape


def test_attention_empty_and_degenerate(A):
    g = gen(4)
    q, k = randn(g, 2, 5, 4, 64, dtype=torch.bfloat16), randn(g, 2, 7, 2, 64, dtype=torch.bfloat16)
    docs = torch.zeros(2, 0, dtype=torch.int32, device="cuda")
    for kk, how in ((k[:, :0], {}), (k[:, :0], dict(documents=docs, causal=True)), (k, dict(lengths=torch.zeros(2, dtype=torch.int32, device="cuda"))),
                    (k, dict(lengths=torch.full((2,), -5, dtype=torch.int32, device="cuda"), causal=True)),
                    (k, dict(causal=True, starts=torch.full((2,), -100, dtype=torch.int32, device="cuda"))),
                    (k, dict(documents=torch.full((2, 7), -1, dtype=torch.int32, device="cuda")))):
        leaves = [t.detach().clone().requires_grad_() for t in (q, kk, kk)]
        o = A.masked_attention(*leaves, **how)
        gr = torch.autograd.grad(o, leaves, torch.ones_like(o))
        assert not any(bool(t.any()) for t in (o,) + gr), how
    leaves = [t.detach().clone().requires_grad_() for t in (q[:, :0], k, k)]
    o = A.masked_attention(*leaves)
    assert o.shape == (2, 0, 4, 64)
    assert not any(bool(t.any()) for t in torch.autograd.grad(o.sum(), leaves))
    assert A.masked_attention(q[:0], k[:0], k[:0]).shape == (0, 5, 4, 64)
    # lengths past the end and starts far away: clamped, and a distance bias from outside the keys is the nearest end's
    far = dict(slopes=torch.full((4,), 0.25, device="cuda"))
    for s, e in ((1 << 30, 6), (-(1 << 30), 0), (2 ** 31 - 1, 6)):
        a = A.masked_attention(q[:, :1], k, k, starts=torch.full((2,), s, dtype=torch.int32, device="cuda"), lengths=torch.full((2,), 1 << 30, dtype=torch.int32, device="cuda"), **far)
        b = A.masked_attention(q[:, :1], k, k, starts=torch.full((2,), e, dtype=torch.int32, device="cuda"), **far)
        assert torch.equal(a, b), s


def test_attention_same_bits_every_run_and_on_other_streams(A):
    q, k, v, do, how = make(ATT_CASES["lengths all"], torch.bfloat16)

    def run():
        leaves = [t.detach().requires_grad_() for t in (q, k, v)]
        o = A.masked_attention(*leaves, **how)
        return (o,) + torch.autograd.grad(o, leaves, do)

    first = run()
    torch.cuda.synchronize()
    streams, results = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams:                                  # three at once
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            results.append(run())
    torch.cuda.synchronize()
    for r in results + [run()]:
        for x, y in zip(first, r):
            assert torch.equal(x, y)


def test_attention_large_offsets(A):
    """A cache whose elements are numbered past 32 bits: only its last sample, at 2^32 elements, is looked at."""
    B, Nk, Hk, D = 9, 1 << 17, 32, 128
    cache = torch.empty(B, Nk, Hk, D, dtype=torch.bfloat16, device="cuda")             # 9.7 GB
    assert cache.stride(0) * (B - 1) >= 1 << 32
    g = gen(8)
    tail = randn(g, Nk, Hk, D, dtype=torch.bfloat16)
    cache[B - 1] = tail
    q = randn(g, B, 1, Hk, D, dtype=torch.bfloat16)
    n = torch.zeros(B, dtype=torch.int32, device="cuda")
    n[B - 1] = Nk
    o = A.masked_attention(q, cache, cache, lengths=n, causal=True)
    assert not bool(o[:B - 1].any())
    assert torch.equal(o[B - 1:], A.masked_attention(q[B - 1:], tail[None], tail[None], causal=True))
    del cache


def test_graph_capture_of_both_operators(A):
    """Norm, rotation and attention as one captured forward, with eager work between the replays; two graphs on one stream's pool."""
    g = gen(11)
    B, N, Hq, Hk, D = 2, 260, 4, 2, 64
    f, pos = A.rope_frequencies(D, device="cuda"), torch.arange(N, device="cuda")
    w = torch.ones(D, device="cuda")
    rows = randn(g, B, N, (Hq + 2 * Hk) * D, dtype=torch.float16)
    docs = ids(g, B, N, 90)
    cache = randn(g, 2, B, 700, Hk, D, dtype=torch.float16)
    n = torch.tensor([700, 333], dtype=torch.int32, device="cuda")

    def whole_row():
        q, k, v = rows.view(B, N, -1, D).split((Hq, Hk, Hk), 2)
        q, k = A.qk_norm_rope(q, k, w, w, pos, f)
        return A.masked_attention(q, k, v, documents=docs, causal=True)

    def step():
        q, _, _ = rows[:, :1].view(B, 1, -1, D).split((Hq, Hk, Hk), 2)
        return A.masked_attention(q, cache[0], cache[1], lengths=n, causal=True, starts=n - 1)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        whole_row(), step()
    torch.cuda.current_stream().wait_stream(s)
    graphs, outs = [], []
    for fn in (whole_row, step):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(fn())
        graphs.append(gr)
    for turn in range(4):
        rows.copy_(randn(g, *rows.shape, dtype=torch.float16))
        for gr in graphs:
            gr.replay()
        eager = [whole_row(), step()]
        torch.cuda.synchronize()
        for x, y in zip(outs, eager):
            assert torch.equal(x, y), turn


def test_graph_capture_of_a_training_step(A):
    """Forward and backward captured together; no eager graph of the same leaves is alive at the capture."""
    g = gen(12)
    B, N, H, D = 1, 200, 2, 64
    f, pos = A.rope_frequencies(D, device="cuda"), torch.arange(N, device="cuda")
    x = [randn(g, B, N, H, D, dtype=torch.bfloat16) for _ in range(3)]
    w = [torch.ones(D, device="cuda") for _ in range(2)]
    do = randn(g, B, N, H, D, dtype=torch.bfloat16)

    def step():
        leaves = [t.detach().requires_grad_() for t in x + w]
        q, k = A.qk_norm_rope(leaves[0], leaves[1], leaves[3], leaves[4], pos, f)
        o = A.masked_attention(q, k, leaves[2], causal=True, softcap=30.0)
        return torch.autograd.grad(o, leaves, do)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = step()
    for turn in range(4):
        for t in x:
            t.copy_(randn(g, *t.shape, dtype=t.dtype))
        gr.replay()
        eager = step()
        torch.cuda.synchronize()
        for a, b in zip(out, eager):
            assert torch.equal(a, b), turn


def test_rotary_attention_layer_end_to_end(A):
    """One projection -> norm and rotation -> attention, forwards and backwards, as a transformer denoiser uses them, against the same in 64 bits;
    then the same rows one token at a time over a cache."""
    g = gen(21)
    B, N, Hq, Hk, D = 2, 96, 4, 2, 64
    dt = torch.bfloat16
    rows = randn(g, B, N, (Hq + 2 * Hk) * D, dtype=dt).requires_grad_()
    wq, wk = (1 + randn(g, D, scale=0.2)).requires_grad_(), (1 + randn(g, D, scale=0.2)).requires_grad_()
    f, pos = A.rope_frequencies(D // 2, device="cuda"), torch.arange(N, device="cuda")
    do = randn(g, B, N, Hq, D, dtype=dt)
    q, k, v = rows.view(B, N, -1, D).split((Hq, Hk, Hk), 2)
    qr, kr = A.qk_norm_rope(q, k, wq, wk, pos, f)
    o = A.masked_attention(qr, kr, v, causal=True)
    grads = torch.autograd.grad(o, (rows, wq, wk), do)
    # every stage against its own statement, on what it was given
    for x, w, y in ((q, wq, qr), (k, wk, kr)):
        within("y", y, O.norm_rope(x.detach(), w.detach(), pos[None], f, 1e-6, False)["y"])
    att = O.attention(qr.detach(), kr.detach(), v.detach(), causal=True, grad=do)
    within("o", o, att["o"])
    leaves = [t.detach().requires_grad_() for t in (qr, kr, v)]
    mid = torch.autograd.grad(A.masked_attention(*leaves, causal=True), leaves, do)
    gq = O.norm_rope(q.detach(), wq.detach(), pos[None], f, 1e-6, False, grad=mid[0])
    gk = O.norm_rope(k.detach(), wk.detach(), pos[None], f, 1e-6, False, grad=mid[1])
    dq, dk, dv = grads[0].view(B, N, -1, D).split((Hq, Hk, Hk), 2)
    within("dq", dq, gq["dx"])
    within("dk", dk, gk["dx"])
    assert torch.equal(dv, mid[2])
    within("dwq", grads[1], gq["dw"])
    within("dwk", grads[2], gk["dw"])
    # one token at a time
    cache = torch.zeros(2, B, N, Hk, D, dtype=dt, device="cuda")
    with torch.no_grad():
        for n in range(N):
            q1, k1 = A.qk_norm_rope(q[:, n:n + 1], k[:, n:n + 1], wq, wk, pos[n:n + 1], f)
            assert torch.equal(q1, qr[:, n:n + 1]) and torch.equal(k1, kr[:, n:n + 1])
            cache[0, :, n:n + 1], cache[1, :, n:n + 1] = k1, v[:, n:n + 1]
            fill = torch.full((B,), n + 1, dtype=torch.int32, device="cuda")
            o1 = A.masked_attention(q1, cache[0], cache[1], causal=True, lengths=fill, starts=fill - 1)
            within(f"token {n}", o1, tuple(t[:, n:n + 1] for t in att["o"]))
