"""Operators of transformer denoisers over token (latent) sequences, on libadk: per-head RMS norm of queries and keys with
the position rotation, and softmax attention with capped scores, a distance bias and causal / prefix / document / length masks.

They take rows ``[B, N, heads, head_dim]`` as a linear projection leaves them (views of one packed projection included) and
carry gradients.  Every call runs on the current stream of its tensors' device; outputs and workspaces come from torch's
allocator on that stream, so a call can be captured in a graph.  No CPU or eager fallback.
"""
import torch
from torch.autograd import forward_ad
from torch.autograd.function import once_differentiable

from . import _lib

__all__ = ["qk_norm_rope", "rope_frequencies", "masked_attention", "alibi_slopes"]

_NORM_TYPES = {torch.float32: _lib.ADK_F32, torch.bfloat16: _lib.ADK_BF16, torch.float16: _lib.ADK_F16}
_ATT_TYPES = {torch.bfloat16: _lib.ADK_BF16, torch.float16: _lib.ADK_F16}
_pack_norm, _pack_att = _lib.packer(_lib.QkNormRopeArgs), _lib.packer(_lib.AttentionArgs)
_LEAST = 2.0 ** -126                   # float32: below lie numbers of fewer bits, and zero
_NO_GRADS = (0,) * 10                  # the backward fields of the norm's struct
_NO_GRAD = (0,) * 7                    # and of the attention's


def _ptr(t):
    return 0 if t is None else t.data_ptr()


def _like(t):
    """New contiguous tensor of t's shape (a third of the time of torch.empty with its type and device)."""
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def rope_frequencies(rotary_dim, base=10000.0, device=None):
    """float64 ``[rotary_dim / 2]`` radians per position: base ** (-2 p / rotary_dim)."""
    if rotary_dim < 0 or rotary_dim % 2:
        raise ValueError(f"rotary_dim {rotary_dim} is not even")
    p = torch.arange(rotary_dim // 2, dtype=torch.float64, device=device)
    return float(base) ** (-2.0 * p / max(rotary_dim, 1))


def alibi_slopes(heads, device=None):
    """float32 ``[heads]`` distance-bias slopes, the geometric series 2 ** (-8 (h + 1) / heads)."""
    return torch.exp2(-8.0 * torch.arange(1, heads + 1, dtype=torch.float64, device=device) / heads).float()


def _on_device(what, device, *tensors):
    if device.type != "cuda":
        raise RuntimeError(f"{what}: tensors are on {device}; there is no CPU path")
    index = device.index
    for t in tensors:
        if t is not None and t.get_device() != index:          # -1 on the CPU
            raise ValueError(f"{what}: tensors on {t.device} and {device}")


def _no_recording(what, *tensors):
    """The library writes through pointers: a forward-mode tangent, or a trace, would be dropped without a word."""
    if forward_ad._current_level >= 0:
        for t in tensors:
            if t is not None and forward_ad.unpack_dual(t).tangent is not None:
                raise NotImplementedError(f"{what}: forward-mode derivatives are not built")
    if torch._C._get_tracing_state() is not None:
        raise NotImplementedError(f"{what}: cannot be recorded by torch.jit.trace")


def _rows(t):
    """Rows as the kernels read them: the elements of a head contiguous (a copy if they are not)."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _rows16(t):
    """Rows with 16-byte aligned heads, at most 2^24 elements apart (a copy if they are not).  The stride of a dimension of one, which a
    slice may leave at anything, does not matter (nor does it to the library, and contiguous() leaves it as it is)."""
    sb, sn, sh, sd = t.stride()
    if sd == 1 and not ((sb | sn | sh) & 7) and sn <= 1 << 24 and not (t.data_ptr() & 15):
        return t
    B, N, H, _ = t.shape
    if sd == 1 and not ((sb * (B > 1) | sn * (N > 1) | sh * (H > 1)) & 7) and (sn <= 1 << 24 or N == 1) and not (t.data_ptr() & 15):
        return t
    t = t.contiguous()
    return t if not (t.data_ptr() & 15) else t.clone()


def _launch(what, device, entry, args, workspace_bytes=None):
    """One library call on the device's current stream; args are its struct's bytes; with workspace_bytes (of the call's arguments)
    also its workspace, from torch's allocator on that stream."""
    if torch._C._cuda_getDevice() != device.index:
        with torch.cuda.device(device):
            return _launch(what, device, entry, args, workspace_bytes)
    stream = torch._C._cuda_getCurrentRawStream(device.index)
    if workspace_bytes is None:
        rc = entry(args, stream)
    elif workspace_bytes > 0:
        w = torch.empty(workspace_bytes, dtype=torch.uint8, device=device)
        rc = entry(args, w.data_ptr(), workspace_bytes, stream)
    else:
        rc = entry(args, None, 0, stream)
    if rc:
        _lib.check(rc, what)


# ---- per-head norm and rotation -------------------------------------------------------------------------------------------

def _norm_args(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved, q_out, k_out, grads=_NO_GRADS):
    """QkNormRopeArgs in the order of its fields; grads: the backward call's."""
    B, N, Hq, D = q.shape
    return _pack_norm(
        _NORM_TYPES[q.dtype], B, N, Hq, k.shape[2], D, 2 * frequencies.shape[0], interleaved, positions.element_size(), eps,
        q.data_ptr(), k.data_ptr(), *q.stride()[:3], *k.stride()[:3],
        _ptr(q_weight), _ptr(k_weight), positions.data_ptr(), *positions.stride(), frequencies.data_ptr(), q_out.data_ptr(), k_out.data_ptr(),
        *grads)


def _norm_forward(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved):
    qo, ko = _like(q), _like(k)
    a = _norm_args(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved, qo, ko)
    _launch("qk_norm_rope", q.device, _lib.load().adk_qk_norm_rope, a)
    return qo, ko


class _QkNormRope(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, q_weight, k_weight, positions, frequencies, eps, interleaved):
        ctx.save_for_backward(q, k, q_weight, k_weight, positions, frequencies)
        ctx.eps, ctx.interleaved = eps, interleaved
        return _norm_forward(q, k, q_weight, k_weight, positions, frequencies, eps, interleaved)

    @staticmethod
    @once_differentiable
    def backward(ctx, gq, gk):
        _no_recording("qk_norm_rope backward", gq, gk)
        q, k, q_weight, k_weight, positions, frequencies = ctx.saved_tensors
        gq, gk = _rows(gq), _rows(gk)
        dq, dk = _like(q), _like(k)
        rows = q.shape[0] * q.shape[1]
        make = torch.empty_like if rows else torch.zeros_like
        dqw = make(q_weight) if q_weight is not None and ctx.needs_input_grad[2] else None
        dkw = make(k_weight) if k_weight is not None and ctx.needs_input_grad[3] else None
        if rows:
            a = _norm_args(q, k, q_weight, k_weight, positions, frequencies, ctx.eps, ctx.interleaved, dq, dk,
                           (gq.data_ptr(), gk.data_ptr(), *gq.stride()[:3], *gk.stride()[:3], _ptr(dqw), _ptr(dkw)))
            lib = _lib.load()
            _launch("qk_norm_rope backward", q.device, lib.adk_qk_norm_rope_backward, a, lib.adk_qk_norm_rope_workspace(a))
        return dq, dk, dqw, dkw, None, None, None, None


def qk_norm_rope(q, k, q_weight, k_weight, positions, frequencies, eps=1e-6, interleaved=False):
    """RMS norm of every head of ``q`` [B, N, Hq, D] and ``k`` [B, N, Hk, D], times the weights, then the rotation of the
    first ``2 * len(frequencies)`` elements by ``positions * frequencies``, in one pass; returns new contiguous (q, k).

    * float32, bfloat16 or float16; D even up to 256; any strides (rows whose elements are not contiguous are copied first).
    * ``q_weight`` / ``k_weight``: [D] of any floating type, or None for ones (computed and differentiated in float32).
    * ``positions``: int32 or int64, [N] or [B, N], any values (expanded views are read as they are).
    * ``frequencies``: float64 [R / 2], radians per position (``rope_frequencies``); may be empty (norm only).
    * ``interleaved``: pairs (2p, 2p + 1) instead of (p, p + R / 2).
    Gradients (reverse mode, once) flow to q, k and the weights, not to positions or frequencies.
    """
    what = "qk_norm_rope"
    if not (q.dim() == 4 and k.dim() == 4 and q.shape[:2] == k.shape[:2] and q.shape[3] == k.shape[3]):
        raise ValueError(f"{what}: q {tuple(q.shape)} and k {tuple(k.shape)} are not [B, N, Hq, D] and [B, N, Hk, D]")
    if not (q.dtype in _NORM_TYPES and k.dtype == q.dtype):
        raise ValueError(f"{what}: q is {q.dtype}, k {k.dtype} (float32, bfloat16 or float16, both alike)")
    B, N, _, D = q.shape
    if not (D % 2 == 0 and 2 <= D <= 256):
        raise ValueError(f"{what}: head dim {D} is not even in [2, 256]")
    if not (q.shape[2] >= 1 and k.shape[2] >= 1):
        raise ValueError(f"{what}: no heads")
    if not (frequencies.dim() == 1 and frequencies.dtype == torch.float64):
        raise ValueError(f"{what}: frequencies must be float64 [R / 2]")
    if not (2 * frequencies.shape[0] <= D):
        raise ValueError(f"{what}: {frequencies.shape[0]} frequencies turn more than the {D} elements of a head")
    if not (positions.dtype in (torch.int32, torch.int64)):
        raise ValueError(f"{what}: positions are {positions.dtype} (int32 or int64)")
    if not (tuple(positions.shape) in ((N,), (B, N))):
        raise ValueError(f"{what}: positions {tuple(positions.shape)} are not [N] or [B, N] = {(B, N)}")
    if not (eps > 0):
        raise ValueError(f"{what}: eps {eps}")
    for w in (q_weight, k_weight):
        if not (w is None or (tuple(w.shape) == (D,) and w.is_floating_point())):
            raise ValueError(f"{what}: a weight is not a floating [{D}]")
    if frequencies.requires_grad:
        raise ValueError(f"{what}: no gradient to frequencies is built")
    _no_recording(what, q, k, q_weight, k_weight, frequencies)
    _on_device(what, q.device, k, q_weight, k_weight, positions, frequencies)
    if positions.dim() == 1:
        positions = positions.expand(B, N)
    q_weight = q_weight.float().contiguous() if q_weight is not None else None
    k_weight = k_weight.float().contiguous() if k_weight is not None else None
    args = (_rows(q), _rows(k), q_weight, k_weight, positions, frequencies.contiguous(), float(eps), int(interleaved))
    if torch.is_grad_enabled() and any(t is not None and t.requires_grad for t in args[:4]):
        return _QkNormRope.apply(*args)
    return _norm_forward(*args)


# ---- attention ------------------------------------------------------------------------------------------------------------

def _att_args(q, k, v, slopes, prefix, documents, lengths, starts, causal, scale, softcap, o, lse, o_low, grads=_NO_GRAD):
    """AttentionArgs in the order of its fields; grads: the backward call's."""
    B, Nq, Hq, D = q.shape
    return _pack_att(
        _ATT_TYPES[q.dtype], B, Nq, k.shape[1], Hq, k.shape[2], D, causal, scale, softcap, q.data_ptr(), k.data_ptr(), v.data_ptr(),
        *q.stride()[:3], *k.stride()[:3], *v.stride()[:3], _ptr(slopes), _ptr(prefix), _ptr(lengths), _ptr(starts), _ptr(documents),
        0 if documents is None else documents.stride(0), o.data_ptr(), _ptr(lse), *grads, _ptr(o_low))


def _att_forward(q, k, v, slopes, prefix, documents, lengths, starts, causal, scale, softcap, lse=None, o_low=None):
    lib = _lib.load()
    o = _like(q)
    a = _att_args(q, k, v, slopes, prefix, documents, lengths, starts, causal, scale, softcap, o, lse, o_low)
    _launch("masked_attention", q.device, lib.adk_attention, a, lib.adk_attention_workspace(a, 0))
    return o


class _MaskedAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, slopes, prefix, documents, lengths, starts, causal, scale, softcap):
        lse = torch.empty((q.shape[0], q.shape[2], q.shape[1]), dtype=torch.float32, device=q.device)
        o_low = _like(q)                   # o in 16 bits more, for the gradient's row sums
        o = _att_forward(q, k, v, slopes, prefix, documents, lengths, starts, causal, scale, softcap, lse, o_low)
        ctx.save_for_backward(q, k, v, slopes, prefix, documents, lengths, starts, o, lse, o_low)
        ctx.how = (causal, scale, softcap)
        return o

    @staticmethod
    @once_differentiable
    def backward(ctx, go):
        _no_recording("masked_attention backward", go)
        q, k, v, slopes, prefix, documents, lengths, starts, o, lse, o_low = ctx.saved_tensors
        dq, dk, dv = _like(q), _like(k), _like(v)
        if q.numel() == 0:
            dk.zero_(), dv.zero_()
        else:
            go = _rows16(go)
            a = _att_args(q, k, v, slopes, prefix, documents, lengths, starts, *ctx.how, o, lse, o_low,
                          (go.data_ptr(), *go.stride()[:3], dq.data_ptr(), dk.data_ptr(), dv.data_ptr()))
            lib = _lib.load()
            _launch("masked_attention backward", q.device, lib.adk_attention_backward, a, lib.adk_attention_workspace(a, 1))
        return dq, dk, dv, None, None, None, None, None, None, None, None


def _index_tensor(what, name, t, shape):
    if not (t.dtype == torch.int32 and tuple(t.shape) == shape):
        raise ValueError(f"{what}: {name} is {t.dtype} {tuple(t.shape)}, must be int32 {list(shape)}")
    return t if t.stride(-1) == 1 or t.shape[-1] <= 1 else t.contiguous()


def masked_attention(q, k, v, *, scale=None, softcap=None, slopes=None, causal=False, prefix=None, documents=None, lengths=None,
                     starts=None):
    """softmax(scores) v for ``q`` [B, Nq, Hq, D], ``k`` and ``v`` [B, Nk, Hk, D]; returns a new contiguous [B, Nq, Hq, D].

    Query head h reads key head h // (Hq // Hk).  Query row i of sample b stands at position p = starts[b] + i (without
    ``starts``: Nk - Nq + i, the last rows of the keys), key j at position j.

    * ``scale``: of the products, default D ** -0.5.  ``softcap`` c: scores become c tanh(score / c), for c up to 1.1e38 (caps over 128
      take a slower form, exact to float32 of the score however small beside the cap).
    * ``slopes`` float32 [Hq]: slopes[h] |p - j| is taken off the scores (``alibi_slopes``; constants, no gradient).
    * ``causal``: row i sees j <= p.  ``prefix`` int32 [B] (with causal): and every j < prefix[b].
    * ``lengths`` int32 [B]: keys j >= lengths[b] do not exist and are not read (values outside [0, Nk] are clamped).
    * ``documents`` int32 [B, Nk]: row i sees keys of its own document, documents[b, p]; negative ids are padding, and
      rows at a position outside [0, Nk) have no document.
    A row that sees nothing gives zeros.  bfloat16 and float16, D = 32, 64 or 128, any strides (rows whose heads are not 16-byte
    aligned are copied first).  Gradients (reverse mode, once) flow to q, k and v, with a fixed summation order.  A single new
    token over a long cache (Nq = 1) is split over the keys.
    """
    what = "masked_attention"
    if not (q.dim() == 4 and k.dim() == 4 and k.shape == v.shape and q.shape[0] == k.shape[0] and q.shape[3] == k.shape[3]):
        raise ValueError(f"{what}: q {tuple(q.shape)}, k {tuple(k.shape)}, v {tuple(v.shape)} are not [B, Nq, Hq, D], [B, Nk, Hk, D] twice")
    if not (q.dtype in _ATT_TYPES and k.dtype == q.dtype and v.dtype == q.dtype):
        raise ValueError(f"{what}: q is {q.dtype}, k {k.dtype}, v {v.dtype} (bfloat16 or float16, all alike)")
    B, Nq, Hq, D = q.shape
    Nk, Hk = k.shape[1:3]
    if not (D in (32, 64, 128)):
        raise ValueError(f"{what}: head dim {D} (32, 64 or 128)")
    if not (Hk >= 1 and Hq >= 1 and Hq % Hk == 0):
        raise ValueError(f"{what}: {Hq} query heads are not a multiple of {Hk} key heads")
    scale = D ** -0.5 if scale is None else float(scale)
    softcap = 0.0 if softcap is None else float(softcap)
    if not (_LEAST <= scale <= 2.3e38):
        raise ValueError(f"{what}: scale {scale} must be in [2^-126, 2.3e38]")
    if not (softcap == 0 or (_LEAST <= softcap <= 1.1e38 and scale <= 1.1e38 * softcap)):
        raise ValueError(f"{what}: softcap {softcap} must be in [2^-126, 1.1e38] and at least scale / 1.1e38 (or None)")
    if not (causal or prefix is None):
        raise ValueError(f"{what}: prefix widens a causal mask: pass causal=True")
    _no_recording(what, q, k, v, slopes)
    _on_device(what, q.device, k, v, slopes, prefix, documents, lengths, starts)
    if slopes is not None:
        if not (slopes.dtype == torch.float32 and tuple(slopes.shape) == (Hq,)):
            raise ValueError(f"{what}: slopes are {slopes.dtype} {tuple(slopes.shape)}, must be float32 [{Hq}]")
        if slopes.requires_grad:
            raise ValueError(f"{what}: slopes are constants; no gradient to them is built")
        slopes = slopes.contiguous()
    prefix = None if prefix is None else _index_tensor(what, "prefix", prefix, (B,))
    lengths = None if lengths is None else _index_tensor(what, "lengths", lengths, (B,))
    starts = None if starts is None else _index_tensor(what, "starts", starts, (B,))
    documents = None if documents is None else _index_tensor(what, "documents", documents, (B, Nk))
    args = (_rows16(q), _rows16(k), _rows16(v), slopes, prefix, documents, lengths, starts, int(causal), scale, softcap)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad):
        return _MaskedAttention.apply(*args)
    return _att_forward(*args)
