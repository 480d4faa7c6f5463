"""Token-sequence operators on the GPU at their edges, against the same 64-bit statements (oracle/token_ops_oracle.py).  Tolerances are
that file's unless a test derives its own."""
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
