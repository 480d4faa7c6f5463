"""Token-sequence operators on the GPU at their edges, against the same 64-bit statements (oracle/token_ops_oracle.py).  Tolerances are
that file's unless a test derives its own."""
import math

import pytest
import torch

from oracle import token_ops_oracle as O
from test_gpu_transformer import A, DT, gen, make, poison, randn, whole, within  # noqa: F401  (A is a fixture)

pytestmark = pytest.mark.gpu


def graded(A, q, k, v, do, **how):
    """(o, dq, dk, dv)"""
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    o = A.masked_attention(*leaves, **how)
    return (o.detach(),) + torch.autograd.grad(o, leaves, do)


# ---- keys that do not exist --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("case", [(2, 300, 300, 2, 2, 64), (6, 300, 300, 16, 4, 128), (3, 1500, 300, 4, 1, 128), (3, 520, 200, 2, 1, 32)],
                         ids=lambda c: "-".join(map(str, c)))
def test_gradients_of_keys_past_the_length_are_zeros(A, case, dt):
    """Infinities and NaN in rows that see nothing (padding: document -1) beside keys past the length, in one block of keys and
    with its rows split over blocks: the gradients of those keys are exact zeros, all others what they are without the poison."""
    B, Nq, Nk, Hq, Hk, D = case
    q, k, v, do, _ = make(case + ({},), DT[dt], seed=6)
    lengths = torch.tensor([Nk - 70, Nk // 2 + 1, 3, 129, 128, Nk], device="cuda", dtype=torch.int32)[:B]
    beyond = torch.arange(Nk, device="cuda")[None] >= lengths[:, None]
    docs = torch.zeros(B, Nk, dtype=torch.int32, device="cuda").masked_fill(beyond, -1)
    g = gen(31)
    if Nq == Nk:
        starts, rows = None, beyond                            # rows past the length are padding
    else:                                                      # and those in front of the keys and behind them
        starts = torch.full((B,), -(Nq - Nk) // 2, device="cuda", dtype=torch.int32)
        p = starts[:, None].long() + torch.arange(Nq, device="cuda")
        rows = (p < 0) | (p >= Nk) | beyond.gather(1, p.clamp(0, Nk - 1))
    for causal in (False, True):
        how = dict(lengths=lengths, documents=docs, causal=causal, starts=starts)
        want = O.attention(q, k, v, grad=do, **how)
        got = graded(A, poison(q, rows, g), poison(k, beyond, g), poison(v, beyond, g), poison(do, rows, g), **how)
        for n, x, clean in (("o", got[0], ~rows), ("dq", got[1], ~rows), ("dk", got[2], ~beyond), ("dv", got[3], ~beyond)):
            within(n, x[clean], tuple(t[clean] for t in want[n]))
        for n, x, none in (("o", got[0], rows), ("dq", got[1], rows), ("dk", got[2], beyond), ("dv", got[3], beyond)):
            assert bool((x[none] == 0).all()), (n, causal)

# ---- capped scores -----------------------------------------------------------------------------------------------------------

CAP_CASES = {
    "step": (3, 1, 900, 8, 2, 128, dict(lengths=True, causal=True, starts=True)),
    "few": (2, 130, 130, 4, 1, 64, dict(causal=True, slopes=True)),
    "few 32": (1, 190, 190, 3, 3, 32, {}),
    "many": (4, 300, 300, 24, 8, 128, dict(causal=True)),
    "many 64": (4, 260, 260, 32, 8, 64, dict(documents=80, causal=True)),
    "many 32": (6, 257, 257, 32, 32, 32, dict(slopes=True)),
    "parts": (1, 1400, 100, 4, 1, 128, {}),
    "query parts": (1, 64, 2200, 4, 2, 64, {}),
}


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("cap", [50.0, 128.0, 129.0, 1e3, 1e5, 1e7, 1e30, 1.1e38])
@pytest.mark.parametrize("name", CAP_CASES)
def test_caps_of_every_size(A, name, cap, dt):
    """Far above the scores a cap does nothing; the error of a capped score belongs to the score, not to the cap."""
    q, k, v, do, how = make(CAP_CASES[name], DT[dt], seed=8)
    how["softcap"] = cap
    want = O.attention(q, k, v, grad=do, **how)
    for n, x in zip(("o", "dq", "dk", "dv"), graded(A, q, k, v, do, **how)):
        within(n, x, want[n])


@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("name", ["step", "few", "many", "many 64", "many 32", "parts"])
def test_scores_of_the_caps_size_beside_small_ones(A, name, dt, monkeypatch):
    """Cap 150; in every second row scores reach it, the rows between keep scores of order one (in the same tiles).  Beside the 1e-4 of
    the products of scores up to 150 (see the oracle) stand 2.4e-7 times the cap from the tanh (its exponential, reciprocal
    and difference, each off by a step of 2^-23 or half of one): 1.4e-4 together, 2e-4 allowed."""
    monkeypatch.setattr(O, "SLACK", 2e-4)
    q, k, v, do, how = make(CAP_CASES[name], DT[dt], seed=9)
    q = q.clone()
    q[:, ::2] *= 16
    how["softcap"] = 150.0
    how.pop("slopes", None)
    want = O.attention(q, k, v, grad=do, **how)
    for n, x in zip(("o", "dq", "dk", "dv"), graded(A, q, k, v, do, **how)):
        within(n, x, want[n])


@pytest.mark.parametrize("cap", [1e-3, 0.5])
def test_small_caps(A, cap):
    q, k, v, do, how = make(CAP_CASES["many 64"], torch.bfloat16, seed=10)
    how["softcap"] = cap
    want = O.attention(q, k, v, grad=do, **how)
    for n, x in zip(("o", "dq", "dk", "dv"), graded(A, q, k, v, do, **how)):
        within(n, x, want[n])



# ---- f16's range -------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("D, Hq, Hk", [(32, 2, 1), (64, 4, 2), (128, 4, 1)])
def test_f16_gradients_of_keys_of_a_quiet_document(A, D, Hq, Hk):
    """Two documents whose gradients are 2^14 apart: the quiet one's are as exact as on their own."""
    N, half = 3000, 1500
    q, k, v, do, _ = make((1, N, N, Hq, Hk, D, {}), torch.float16, seed=11)
    docs = (torch.arange(N, device="cuda") >= half).int()[None]
    mix = (torch.arange(N, device="cuda") % 3 == 1).int()[None]                # taking turns: both in every tile
    for d in (docs, mix):
        g = torch.where(d[..., None, None] == 0, do * 2.0 ** 10, do * 2.0 ** -4)
        got = graded(A, q, k, v, g, documents=d)
        for which in (0, 1):
            at = d[0] == which
            want = O.attention(*(t[:, at] for t in (q, k, v)), grad=g[:, at])
            for n, x in zip(("o", "dq", "dk", "dv"), got):
                within(f"{n} of document {which}", x[:, at], want[n])


@pytest.mark.parametrize("D", [32, 64, 128])
def test_f16_gradients_of_keys_that_only_quiet_rows_see(A, D):
    """Causal: the last rows' gradients are 2^14 smaller than the first ones', and the last keys are seen by those alone."""
    N, half = 1100, 700
    q, k, v, do, _ = make((1, N, N, 4, 2, D, {}), torch.float16, seed=12)
    quiet = (torch.arange(N, device="cuda") >= half)[None, :, None, None]
    g = torch.where(quiet, do * 2.0 ** -4, do * 2.0 ** 10)
    got = graded(A, q, k, v, g, causal=True)
    want = O.attention(q, k, v, grad=g, causal=True)
    for n, x in zip(("o", "dq", "dk", "dv"), got):
        within(n, x, want[n])
    alone = O.attention(q, k, v, grad=torch.where(quiet, g, 0.0), causal=True)
    for n, x in zip(("dk", "dv"), got[2:]):
        within(f"{n} of the last keys", x[:, half:], tuple(t[:, half:] for t in alone[n]))


@pytest.mark.parametrize("scale", [2.0 ** -10, 1.0, 1000.0])
@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("case", [(2, 260, 260, 8, 2, 64), (2, 300, 300, 4, 1, 128)], ids=lambda c: "-".join(map(str, c)))
def test_gradients_of_other_sizes(A, case, dt, scale):
    q, k, v, do, how = make(case + (dict(causal=True, documents=90),), DT[dt], seed=13)
    do = do * scale
    want = O.attention(q, k, v, grad=do, **how)
    for n, x in zip(("o", "dq", "dk", "dv"), graded(A, q, k, v, do, **how)):
        within(n, x, want[n])



@pytest.mark.parametrize("case", [(1, 1, 1 << 17, 2, 1, 64), (1, 2048, 1 << 16, 4, 1, 64), (1, 2048, 1 << 16, 12, 1, 128)], ids=lambda c: "-".join(map(str, c)))
def test_f16_many_small_probabilities(A, case):
    """One key holds nearly all, the others 2^-25 of it each, and only they have values.  A probability is rounded to f16's step of 2^-24
    at most after it was taken relative to 2^-7 of the largest: 2^-32 is the largest error of each, not 2^-25."""
    B, Nq, Nk, Hq, Hk, D = case
    q = torch.zeros(B, Nq, Hq, D, dtype=torch.float16, device="cuda")
    k = torch.zeros(B, Nk, Hk, D, dtype=torch.float16, device="cuda")
    v = torch.ones(B, Nk, Hk, D, dtype=torch.float16, device="cuda")
    q[..., 0] = 1.0
    k[:, Nk // 3, :, 0] = 25.0
    v[:, Nk // 3] = 0.0
    o = A.masked_attention(q, k, v, scale=math.log(2.0)).double()
    rest = (Nk - 1) * 2.0 ** -25
    want = rest / (1 + rest)
    assert float((o - want).abs().max()) <= (1e-4 + 2.0 ** -10) * want + Nk * 2.0 ** -32, (float(o.min()), float(o.max()), want)


# ---- far keys ----------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("Nq, Hq", [(1, 2), (130, 2), (2048, 16)])
def test_distances_behind_2_to_the_24th_key(A, Nq, Hq):
    """Distances of a bias are whole numbers up to rounding of the DISTANCE, wherever the keys stand."""
    Nk, D, tail = (1 << 24) + 4099, 32, 2048 + 512
    g = gen(14)
    q, do = randn(g, 1, Nq, Hq, D, dtype=torch.bfloat16), randn(g, 1, Nq, Hq, D, dtype=torch.bfloat16)
    kt, vt = randn(g, 1, tail, 1, D, dtype=torch.bfloat16), randn(g, 1, tail, 1, D, dtype=torch.bfloat16)
    k = torch.zeros(1, Nk, 1, D, dtype=torch.bfloat16, device="cuda")
    v = torch.zeros(1, Nk, 1, D, dtype=torch.bfloat16, device="cuda")
    k[:, Nk - tail:], v[:, Nk - tail:] = kt, vt
    docs = torch.full((1, Nk), -1, dtype=torch.int32, device="cuda")
    docs[:, Nk - tail:] = 3
    slopes = torch.linspace(0.3, 1.5, Hq, device="cuda")
    for causal in (True, False):
        want = O.attention(q, kt, vt, grad=do, slopes=slopes, causal=causal)       # the tail alone
        got = graded(A, q, k, v, do, slopes=slopes, causal=causal, documents=docs)
        for n, x in zip(("o", "dq", "dk", "dv"), got):
            within(n, x[:, Nk - tail:] if n in ("dk", "dv") else x, want[n])


# ---- what is not built --------------------------------------------------------------------------------------------------------

def test_tangents_of_gradients_are_refused(A):
    q, k, v, do, _ = make((1, 20, 20, 2, 1, 64, {}), torch.bfloat16)
    leaves = [t.detach().requires_grad_() for t in (q, k, v)]
    f, pos = A.rope_frequencies(64, device="cuda"), torch.arange(20, device="cuda")
    o, y = A.masked_attention(*leaves), A.qk_norm_rope(leaves[0], leaves[1], None, None, pos, f)[0]
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(do, torch.ones_like(do))
        for out in (o, y):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                torch.autograd.grad(out, leaves[0], dual, retain_graph=True)
        assert all(bool(torch.isfinite(g).all()) for g in torch.autograd.grad(o, leaves, do))      # a plain gradient passes


# ---- views ---------------------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("shape", [(1, 150, 150, 4, 2), (1, 1, 900, 8, 2), (2, 1, 1, 4, 1), (1, 40, 40, 1, 1), (3, 1, 70, 1, 1), (1, 300, 1, 2, 1)], ids=lambda c: "-".join(map(str, c)))
def test_views_with_odd_strides_of_dimensions_of_one(A, shape):
    """One sample of a padded buffer, one token, one head: the same bits as contiguous tensors; the incoming gradient too."""
    B, Nq, Nk, Hq, Hk = shape
    q, k, v, do, _ = make((B, Nq, Nk, Hq, Hk, 64, {}), torch.bfloat16, seed=16)

    def odd(t):
        """t with the strides of its dimensions of one set to 67."""
        return t.as_strided(t.shape, [67 if n == 1 else s for n, s in zip(t.shape, t.stride())])

    assert any(s == 67 for t in (q, k, do) for s in odd(t).stride())
    base = graded(A, q, k, v, do, causal=True)
    leaves = [odd(t).detach().requires_grad_() for t in (q, k, v)]
    o = A.masked_attention(*leaves, causal=True)
    for x, y in zip(base, (o,) + torch.autograd.grad(o, leaves, odd(do))):
        assert torch.equal(x, y)
    for x, y in zip(base, graded(A, *(odd(t) for t in (q, k, v, do)), causal=True)):
        assert torch.equal(x, y)


def test_an_empty_cache_with_odd_strides(A):
    q = torch.ones(2, 3, 2, 64, dtype=torch.float16, device="cuda")
    k = torch.ones(2, 5, 2, 67, dtype=torch.float16, device="cuda")[:, :0, :, 1:65]
    got = graded(A, q, k, k, q, causal=True)
    assert got[2].shape == (2, 0, 2, 64) and not any(bool(t.any()) for t in got)


# ---- sizes ---------------------------------------------------------------------------------------------------------------------

def test_norm_of_more_rows_than_one_row_of_the_grid_holds(A):
    """2^26 tokens are 2^32 threads."""
    N = (1 << 26) + 5
    q = torch.zeros(1, N, 1, 2, dtype=torch.bfloat16, device="cuda")
    g = gen(17)
    for at in (0, (1 << 24) - 3, N - 300):                    # the first, where a row of the grid ends, the last
        q[:, at:at + 300] = randn(g, 1, 300, 1, 2, dtype=torch.bfloat16)
    f, pos = A.rope_frequencies(2, device="cuda"), torch.arange(N, device="cuda")
    y, z = A.qk_norm_rope(q, q, None, None, pos, f)
    for at in (0, (1 << 24) - 3, N - 300):
        part = q[:, at:at + 300].contiguous()
        assert torch.equal(y[:, at:at + 300], A.qk_norm_rope(part, part, None, None, pos[at:at + 300], f)[0])
    assert torch.equal(y, z)


# ---- a scale of one's own ------------------------------------------------------------------------------------------------------


def test_gradients_with_offsets_past_2_to_the_31st(A):
    """Rows, and keys, whose elements are numbered past 2^31: only the last of them have values; every other gradient is zero."""
    D, tail, few = 64, 200, 70
    long = (1 << 25) + 37                                     # 2^31 elements of 64
    g = gen(18)

    def behind(t):
        wide = torch.zeros(1, long, 1, D, dtype=torch.bfloat16, device="cuda")
        wide[:, long - tail:] = t
        return wide

    a, b, c = (randn(g, 1, tail, 1, D, dtype=torch.bfloat16) for _ in range(3))
    x, y, z = (randn(g, 1, few, 1, D, dtype=torch.bfloat16) for _ in range(3))
    # many rows, few keys; dO of the rows without values is zero, so they add nothing to dK and dV
    want = O.attention(a, x, y, grad=b)
    o, dq, dk, dv = graded(A, behind(a), x, y, behind(b))
    for n, got in (("o", o[:, long - tail:]), ("dq", dq[:, long - tail:]), ("dk", dk), ("dv", dv)):
        within(n, got, want[n])
    assert not bool(dq[:, :long - tail].any())
    del o, dq, dk, dv
    # few rows, many keys: a document holds the last of them
    docs = torch.full((1, long), -1, dtype=torch.int32, device="cuda")
    docs[:, long - tail:] = 1
    want = O.attention(x, a, b, grad=z)
    o, dq, dk, dv = graded(A, x, behind(a), behind(b), z, documents=docs)
    for n, got in (("o", o), ("dq", dq), ("dk", dk[:, long - tail:]), ("dv", dv[:, long - tail:])):
        within(n, got, want[n])
    assert not bool(dk[:, :long - tail].any()) and not bool(dv[:, :long - tail].any())


@pytest.mark.parametrize("D", [32, 64, 128])
def test_f16_quiet_gradients_beside_infinite_ones_of_padding(A, D):
    """Infinities and NaN in rows that see nothing take no part in the scale of the others' gradients (2^-8)."""
    N = 700
    q, k, v, do, _ = make((2, N, N, 4, 2, D, {}), torch.float16, seed=19)
    docs = (torch.arange(N, device="cuda") * 7 // N).int().repeat(2, 1)
    docs[:, 5::9] = -1                                       # padding in every tile
    rows, do = docs < 0, do * 2.0 ** -8
    want = O.attention(q, k, v, grad=do, documents=docs, causal=True)
    g = gen(20)
    got = graded(A, poison(q, rows, g), poison(k, rows, g), poison(v, rows, g), poison(do, rows, g), documents=docs, causal=True)
    for n, x in zip(("o", "dq", "dk", "dv"), got):
        within(n, x[~rows], tuple(t[~rows] for t in want[n]))
        assert bool((x[rows] == 0).all()), n


@pytest.mark.parametrize("softcap", [None, 30.0, 1e4])
def test_graph_capture_of_f16_gradients(A, softcap):
    """Forward and backward with all of f16's scratch captured; every replay against the eager result."""
    g = gen(22)
    x = [randn(g, 2, 300, 4, 64, dtype=torch.float16) for _ in range(4)]
    docs = torch.cumsum(torch.rand(2, 300, generator=g, device="cuda") < 0.02, 1).int()

    def step():
        return graded(A, *x, documents=docs, causal=True, softcap=softcap)

    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    gr = torch.cuda.CUDAGraph()
    with torch.cuda.graph(gr):
        out = step()
    for turn in range(4):
        for n, t in enumerate(x):
            t.copy_(randn(g, *t.shape, dtype=t.dtype, scale=4.0 ** (turn - 2) if n == 3 else 1.0))
        gr.replay()
        eager = step()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, eager)), turn


# ---- precision of the gradients --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dt", ["bf16", "f16"])
@pytest.mark.parametrize("case", [(1, 300, 900, 4, 2, 64), (6, 300, 900, 16, 4, 128), (1, 8, 2500, 2, 1, 32)], ids=lambda c: "-".join(map(str, c)))
def test_gradients_of_scores_of_nearly_equal_values(A, case, dt):
    """v is one row for all keys and a 2^-6 of noise, so that dP - delta is a small difference of large numbers.  Rounding o alone would
    put delta off by a third of half a step of the common row, 0.3 u 2^6 of the difference: 4 % in bf16, 0.5 % in f16.  What remains: the rounding of
    the probabilities in the forward, which the n keys average to 0.6 u 2^6 / sqrt(n) (0.25 %, 0.03 %), of dS and of the result (0.6 u each).
    Four times that is allowed, of the norm."""
    B, Nq, Nk, Hq, Hk, D = case
    q, k, v, do, _ = make(case + ({},), DT[dt], seed=23, scale=0.5)
    g = gen(24)
    v = (randn(g, B, 1, Hk, D) + 2.0 ** -6 * v.float()).to(DT[dt])
    want = O.attention(q, k, v, grad=do)
    got = graded(A, q, k, v, do)
    u = torch.finfo(DT[dt]).eps / 2
    bound = 4 * (0.6 * u * 64 / Nk ** 0.5 + 2 * 0.6 * u)
    for n, x in zip(("dq", "dk"), got[1:3]):
        value = want[n][0]
        off = float((x.double() - value).norm() / value.norm())
        assert off <= bound, (n, off, bound)
