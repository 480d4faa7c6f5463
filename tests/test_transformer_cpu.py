"""CPU: what the token-sequence operators refuse, in the C ABI (before anything is launched) and in Python, their workspace sizes, and
the structs' mirrors.  Pointers below are never followed."""
import ctypes as C

import pytest
import torch

import audio_diffusion_amd as A
from audio_diffusion_amd import _lib

P = 4096                                                     # a 16-byte aligned address that nothing reads


def norm_args(**kw):
    a = _lib.QkNormRopeArgs()
    a.dtype, a.B, a.N, a.Hq, a.Hk, a.D, a.R, a.pos_bytes, a.eps = 1, 2, 3, 4, 2, 64, 32, 8, 1e-6
    a.q = a.k = a.q_out = a.k_out = a.positions = a.frequencies = a.q_grad = a.k_grad = P
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def att_args(**kw):
    a = _lib.AttentionArgs()
    a.dtype, a.B, a.Nq, a.Nk, a.Hq, a.Hk, a.D, a.scale = 1, 2, 30, 40, 4, 2, 64, 0.125
    a.q = a.k = a.v = a.o = a.lse = a.o_grad = a.q_grad = a.k_grad = a.v_grad = P
    a.q_stride_b, a.q_stride_n, a.q_stride_h = 30 * 256, 256, 64
    a.k_stride_b, a.k_stride_n, a.k_stride_h = 40 * 128, 128, 64
    a.v_stride_b, a.v_stride_n, a.v_stride_h = 40 * 128, 128, 64
    a.og_stride_b, a.og_stride_n, a.og_stride_h = 30 * 256, 256, 64
    for n, v in kw.items():
        setattr(a, n, v)
    return a


def refused(rc, words):
    assert rc == -1
    text = _lib.load().adk_last_error().decode()
    assert words in text, text


def test_struct_sizes():
    lib = _lib.load()
    assert lib.adk_sizeof_qk_norm_rope() == C.sizeof(_lib.QkNormRopeArgs)
    assert lib.adk_sizeof_attention() == C.sizeof(_lib.AttentionArgs)


@pytest.mark.parametrize("kw, words", [
    (dict(dtype=7), "dtype"), (dict(B=-1), "B=-1"), (dict(B=1 << 20, N=1 << 20), "2^31"), (dict(Hq=0), "heads"), (dict(Hk=1 << 20), "heads"),
    (dict(D=65), "head dim"), (dict(D=258), "head dim"), (dict(D=0), "head dim"), (dict(R=33), "R=33"), (dict(R=66), "R=66"), (dict(R=-2), "R=-2"),
    (dict(eps=0.0), "eps"), (dict(eps=float("nan")), "eps"), (dict(pos_bytes=2), "positions"), (dict(q=None), "null"), (dict(positions=None), "null"),
    (dict(frequencies=None), "null"), (dict(k_out=None), "null"), (dict(q=P + 1), "aligned"), (dict(dtype=0, k=P + 2), "aligned")])
def test_norm_refusals(kw, words):
    lib = _lib.load()
    refused(lib.adk_qk_norm_rope(C.byref(norm_args(**kw)), None), words)
    refused(lib.adk_qk_norm_rope_backward(C.byref(norm_args(**kw)), C.c_void_p(P), 1 << 40, None), words)


def test_norm_backward_refusals_and_workspace():
    lib = _lib.load()
    need = lib.adk_qk_norm_rope_workspace(C.byref(norm_args()))
    assert need > 0 and lib.adk_qk_norm_rope_workspace(C.byref(norm_args(D=3))) == -1
    refused(lib.adk_qk_norm_rope_backward(C.byref(norm_args()), None, need, None), "workspace")
    refused(lib.adk_qk_norm_rope_backward(C.byref(norm_args()), C.c_void_p(P), need - 1, None), "workspace")
    refused(lib.adk_qk_norm_rope_backward(C.byref(norm_args()), C.c_void_p(P + 4), need, None), "workspace")
    refused(lib.adk_qk_norm_rope_backward(C.byref(norm_args(q_grad=None)), C.c_void_p(P), need, None), "gradient")
    refused(lib.adk_qk_norm_rope_backward(C.byref(norm_args(B=0, q_weight_grad=P)), C.c_void_p(P), need, None), "weight gradient")
    refused(lib.adk_qk_norm_rope(None, None), "null")
    # nothing to do is no error, and nothing is read
    assert lib.adk_qk_norm_rope(C.byref(norm_args(B=0, q=None)), None) == 0
    assert lib.adk_qk_norm_rope_backward(C.byref(norm_args(N=0, q=None)), None, 0, None) == 0


@pytest.mark.parametrize("kw, words", [
    (dict(dtype=0), "dtype"), (dict(dtype=5), "dtype"), (dict(D=48), "head dim"), (dict(D=256), "head dim"), (dict(Hq=3), "multiple"), (dict(Hk=0), "multiple"),
    (dict(Nq=-1), "Nq"), (dict(Nk=(1 << 28) + 1), "2^28"), (dict(B=70000), "grid"), (dict(B=60000, Hq=4096, Hk=4096, Nq=32000), "grid"),
    (dict(scale=0.0), "scale"), (dict(scale=float("inf")), "scale"), (dict(scale=float("nan")), "scale"), (dict(softcap=-1.0), "softcap"),
    (dict(softcap=float("nan")), "softcap"), (dict(prefix=P), "prefix"), (dict(q=None), "null"), (dict(v=None), "null"), (dict(o=None), "null"),
    (dict(k=P + 2), "aligned"), (dict(o=P + 8), "aligned"), (dict(k_stride_h=60), "strides"), (dict(q_stride_n=(1 << 24) + 8), "2^24"), (dict(v_stride_n=-128), "2^24")])
def test_attention_refusals(kw, words):
    lib = _lib.load()
    refused(lib.adk_attention(C.byref(att_args(**kw)), C.c_void_p(P), 1 << 40, None), words)
    refused(lib.adk_attention_backward(C.byref(att_args(**kw)), C.c_void_p(P), 1 << 40, None), words)


def test_attention_backward_refusals_and_workspaces():
    lib = _lib.load()
    assert lib.adk_attention_workspace(C.byref(att_args()), 0) == 0
    docs = att_args(documents=P, documents_stride=40)
    assert lib.adk_attention_workspace(C.byref(docs), 0) == 256
    refused(lib.adk_attention(C.byref(docs), None, 0, None), "workspace")
    # a long cache is split: f32 partial sums of every row and split
    split = att_args(Nq=1, Nk=65536, B=1, Hq=8, Hk=2)
    n = lib.adk_attention_workspace(C.byref(split), 0)
    assert n > 0 and n % (8 * (64 + 2) * 4) == 0
    refused(lib.adk_attention(C.byref(split), C.c_void_p(P), n - 1, None), "workspace")
    need = lib.adk_attention_workspace(C.byref(att_args()), 1)
    assert need >= 2 * 4 * 30 * 4
    for kw, words in ((dict(lse=None), "null"), (dict(o_grad=None), "null"), (dict(k_grad=None), "null"), (dict(o_grad=P + 2), "aligned"), (dict(og_stride_n=4), "aligned"),
                      (dict(og_stride_n=1 << 25), "2^24"), (dict(Nq=0), "no query rows")):
        refused(lib.adk_attention_backward(C.byref(att_args(**kw)), C.c_void_p(P), need, None), words)
    refused(lib.adk_attention_backward(C.byref(att_args()), C.c_void_p(P), need - 1, None), "workspace")
    refused(lib.adk_attention(None, None, 0, None), "null")
    assert lib.adk_attention_workspace(C.byref(att_args(D=1)), 0) == -1
    for kw in (dict(B=0), dict(Nq=0)):
        assert lib.adk_attention(C.byref(att_args(q=None, **kw)), None, 0, None) == 0
        assert lib.adk_attention_workspace(C.byref(att_args(**kw)), 0) >= 0
    assert lib.adk_attention_backward(C.byref(att_args(B=0)), None, 0, None) == 0


def qkv(B=2, Nq=3, Nk=5, Hq=4, Hk=2, D=64, dtype=torch.bfloat16):
    return torch.zeros(B, Nq, Hq, D, dtype=dtype), torch.zeros(B, Nk, Hk, D, dtype=dtype), torch.zeros(B, Nk, Hk, D, dtype=dtype)


def test_python_refusals_attention():
    q, k, v = qkv()
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)                        # noqa: E731
    with pytest.raises(RuntimeError, match="no CPU path"):
        A.masked_attention(q, k, v)
    for args, kw, words in (((q[0], k, v), {}, "are not"), ((q, k, v[:, :4]), {}, "are not"), ((q, k[..., :32], v[..., :32]), {}, "are not"),
                            ((q.float(), k.float(), v.float()), {}, "float32"), ((q, k.half(), v), {}, "alike"), (qkv(D=48), {}, "head dim"), (qkv(Hq=3), {}, "multiple"),
                            ((q, k, v), dict(scale=-1.0), "scale"), ((q, k, v), dict(scale=float("nan")), "scale"), ((q, k, v), dict(softcap=-2), "softcap"),
                            ((q, k, v), dict(prefix=i32(2)), "causal")):
        with pytest.raises(ValueError, match=words):
            A.masked_attention(*args, **kw)


def test_python_refusals_norm():
    q, k, _ = qkv(Nk=3)
    pos, f = torch.arange(3), A.rope_frequencies(64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        A.qk_norm_rope(q, k, None, None, pos, f)
    w = torch.ones(64)
    for args, kw, words in (((q, k[:, :2], None, None, pos, f), {}, "are not"), ((q.double(), k.double(), None, None, pos, f), {}, "float64"),
                            ((q, k.half(), None, None, pos, f), {}, "alike"), ((q, k, None, None, pos.float(), f), {}, "positions"),
                            ((q, k, None, None, pos[:2], f), {}, "positions"), ((q, k, None, None, pos, f.float()), {}, "float64"),
                            ((q, k, None, None, pos, A.rope_frequencies(66)), {}, "more than"), ((q, k, w[:5], None, pos, f), {}, "weight"),
                            ((q, k, None, w.int(), pos, f), {}, "weight"), ((q, k, None, None, pos, f), dict(eps=0), "eps"),
                            ((q, k, None, None, pos, f.clone().requires_grad_()), {}, "frequencies")):
        with pytest.raises(ValueError, match=words):
            A.qk_norm_rope(*args, **kw)
    with pytest.raises(ValueError):
        A.rope_frequencies(7)


def test_frequencies_and_slopes():
    f = A.rope_frequencies(8, base=100.0)
    assert f.dtype == torch.float64 and torch.allclose(f, torch.tensor([1.0, 100 ** -0.25, 0.1, 100 ** -0.75], dtype=torch.float64))
    assert A.rope_frequencies(0).numel() == 0
    s = A.alibi_slopes(4)
    assert s.dtype == torch.float32 and s.tolist() == [0.25, 0.0625, 0.015625, 0.00390625]


def test_packed_structs_have_the_mirrors_layout_and_cut_nothing_off():
    for mirror in (_lib.QkNormRopeArgs, _lib.AttentionArgs):
        pack = _lib.packer(mirror)
        values = [float(n + 1) if t is C.c_float else n + 1 for n, (_, t) in enumerate(mirror._fields_)]
        a = mirror.from_buffer_copy(pack(*values))
        assert [getattr(a, name) for name, _ in mirror._fields_] == values
        for n, (_, t) in enumerate(mirror._fields_):
            if t in (C.c_int32, C.c_float):
                with pytest.raises(ValueError, match="beyond"):
                    pack(*values[:n], 1 << 31 if t is C.c_int32 else 1e39, *values[n + 1:])


@pytest.mark.parametrize("kw", [dict(softcap=1.2e38), dict(softcap=3e38), dict(softcap=1e-39), dict(scale=2.4e38), dict(scale=1e30, softcap=1e-9)])
def test_scores_outside_the_range_of_f32_are_refused(kw):
    lib = _lib.load()
    refused(lib.adk_attention(C.byref(att_args(**kw)), C.c_void_p(P), 1 << 40, None), "range")
    refused(lib.adk_attention_backward(C.byref(att_args(**kw)), C.c_void_p(P), 1 << 40, None), "range")
    for ok in (dict(softcap=1.1e38), dict(softcap=1e-30), dict(scale=2.3e38), dict(scale=1e-30)):
        assert lib.adk_attention_workspace(C.byref(att_args(**ok)), 0) >= 0


@pytest.mark.parametrize("kw", [dict(softcap=1e-50), dict(softcap=1e-46), dict(scale=1e-50)])
def test_a_cap_or_scale_that_f32_does_not_have_is_refused(kw):
    """and is not taken for no cap."""
    with pytest.raises(ValueError, match=next(iter(kw))):
        A.masked_attention(*qkv(), **kw)


def test_forward_mode_tangents_and_traces_are_refused_not_dropped():
    """(Before the tensors' device is looked at.)  Plain tensors inside a dual level pass on to the next check."""
    q, k, v = qkv(Nk=3)
    pos, f, w, s = torch.arange(3), A.rope_frequencies(64), torch.ones(64), torch.ones(4)
    with torch.autograd.forward_ad.dual_level():
        dual = lambda t: torch.autograd.forward_ad.make_dual(t, torch.ones_like(t))          # noqa: E731
        for args in ((dual(q), k, v), (q, dual(k), v), (q, k, dual(v))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                A.masked_attention(*args)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            A.masked_attention(q, k, v, slopes=dual(s))
        for args in ((dual(q), k, w, w, pos, f), (q, dual(k), w, w, pos, f), (q, k, dual(w), w, pos, f), (q, k, w, dual(w), pos, f), (q, k, w, w, pos, dual(f))):
            with pytest.raises(NotImplementedError, match="forward-mode"):
                A.qk_norm_rope(*args)
        with pytest.raises(RuntimeError, match="no CPU path"):
            A.masked_attention(q, k, v)
        with pytest.raises(RuntimeError, match="no CPU path"):
            A.qk_norm_rope(q, k, w, w, pos, f)
    for fn, args in ((A.masked_attention, (q, k, v)), (lambda q, k: A.qk_norm_rope(q, k, w, w, pos, f), (q, k))):
        with pytest.raises(NotImplementedError, match="trace"):
            torch.jit.trace(fn, args)


def test_strides_of_dimensions_of_one_do_not_matter():
    """Views that torch calls contiguous whatever the stride of a dimension of one: nothing is copied, nothing refused."""
    from audio_diffusion_amd import transformer as T
    bf = torch.bfloat16
    for t in (torch.zeros(2, 643, dtype=bf)[:, :640].view(2, 5, 2, 64)[:1],                  # one sample of a padded buffer
              torch.zeros(1, 6, 1, 67, dtype=bf)[:, :1, :, :64],                              # one token of one padded head
              torch.zeros(2, 3, 67, 64, dtype=bf).transpose(1, 2)[:, :, 1:2][:1, :1],
              torch.zeros(1, 1, 1, (1 << 24) + 64, dtype=bf)[..., :64].expand(3, 1, 1, 64)):
        assert T._rows16(t) is t, t.stride()
        assert t.shape[-1] == 64
    odd = torch.zeros(2, 643, dtype=bf)[:, :640].view(2, 5, 2, 64)                            # two samples: copied
    assert T._rows16(odd) is not odd and T._rows16(odd).stride() == (640, 128, 64, 1)
    lib = _lib.load()
    docs = dict(documents=P, documents_stride=40)                                             # a call that needs a workspace: refused for that alone
    for kw in (dict(B=1, q_stride_b=643, k_stride_b=3, v_stride_b=-5, og_stride_b=1), dict(Nq=1, q_stride_n=67, og_stride_n=-3), dict(Nq=1, q_stride_n=1 << 30),
               dict(Hq=1, Hk=1, q_stride_h=67, k_stride_h=67, v_stride_h=1, og_stride_h=9), dict(Nk=1, k_stride_n=67, v_stride_n=1 << 40),
               dict(Nk=0, k=P + 2, v=P + 2, k_stride_b=3, v_stride_h=5, k_stride_n=-7)):
        if kw.get("Nk") != 0:                                                                 # (no keys: no ranges of documents)
            refused(lib.adk_attention(C.byref(att_args(**docs, **kw)), None, 0, None), "workspace")
        refused(lib.adk_attention_backward(C.byref(att_args(**docs, **kw)), None, 0, None), "workspace")
        refused(lib.adk_attention_backward(C.byref(att_args(**docs, **dict(kw, Nq=2, B=2, Hq=2, Hk=2, Nk=2, k=P, v=P))), None, 0, None), "stride")


def test_launches_of_more_threads_than_there_can_be_are_refused():
    """2^32 threads are the end; what stays below reaches the next check."""
    lib = _lib.load()
    docs = dict(documents=P, documents_stride=40)
    for kw in (dict(B=65535, Hq=512, Hk=512, Nq=1), dict(B=65535, Hq=512, Hk=1, Nq=64), dict(B=65535, Hq=32, Hk=8, Nq=5000)):
        refused(lib.adk_attention(C.byref(att_args(**kw, **docs)), None, 0, None), "grid")
    for kw in (dict(B=65535, Hq=256, Hk=128, Nq=1), dict(B=65535, Hq=32, Hk=8, Nq=1), dict(B=1, Hq=8, Hk=8, Nq=1 << 20)):
        refused(lib.adk_attention(C.byref(att_args(**kw, **docs)), None, 0, None), "workspace")
    for kw in (dict(B=65535, Hq=256, Hk=128, Nq=1), dict(B=65535, Hq=8, Hk=8, Nk=5000)):
        refused(lib.adk_attention_backward(C.byref(att_args(**kw, **docs)), None, 0, None), "grid")
    # few rows over a very long cache: the partial sums stay below 1.2 GB whatever its length
    for Nk in (1 << 20, 1 << 24, 1 << 28):
        assert 0 < lib.adk_attention_workspace(C.byref(att_args(B=1, Hq=8, Hk=8, Nq=2040, Nk=Nk, D=128)), 0) < 1.2e9
