"""Operator API mirroring the reference's hot-path Metal kernels.

    relu2(x)                        metal_kernels.py:37-47,62-68
    rope_ht(x, cs, sn, pos0=0)      metal_kernels.py:87-134
    make_rope_tables(T, D, base)    metal_kernels.py:144-150
    rms(x)                          model.py:48-49
    qk_norm_rope(q, k, cs, sn)      rms and rope_ht of q and k in one pass
                                    (model.py:244-247); qk_norm_rope_bwd is its gradient
    sample_logits(logits, u, ...)   sample.py:45-49 by given random numbers, with
                                    top_p and min_p

Inputs are torch tensors on the GPU (fp32 or bf16); outputs keep the input
dtype, computed in fp32 inside the HIP kernels.  ``rope_ht`` takes the
position of row 0 explicitly (the reference derives it from the row index
within the tensor, i.e. pos0 = 0).
"""

import ctypes

import torch

from . import _lib
from ._stream import current_stream, on_device


def _dt(x):
    if x.dtype == torch.float32:
        return _lib.DTYPE_F32
    if x.dtype == torch.bfloat16:
        return _lib.DTYPE_BF16
    raise TypeError(f"unsupported dtype {x.dtype} (float32 or bfloat16)")


def _gpu(x):
    if not (isinstance(x, torch.Tensor) and x.is_cuda):
        raise ValueError("expected a GPU tensor")
    return x.contiguous()


def _p(t):
    return ctypes.c_void_p(t.data_ptr())


def relu2(x):
    x = _gpu(x)
    y = torch.empty_like(x)
    _lib.check(_lib.lib().ann_op_relu2(_p(x), _p(y), x.numel(), _dt(x), current_stream()))
    return y


def rope_ht(x, cs, sn, pos0=0, inverse=False):
    x = _gpu(x)
    cs, sn = _gpu(cs).float(), _gpu(sn).float()
    if x.dim() != 4:
        raise ValueError("x must be (B, T, H, D)")
    B, T, H, D = x.shape
    if cs.shape[-1] != D // 4 or cs.shape[0] < pos0 + T or sn.shape != cs.shape:
        raise ValueError("tables must be (>= pos0 + T, D/4)")
    y = torch.empty_like(x)
    _lib.check(_lib.lib().ann_op_rope_ht(_p(x), _p(y), _p(cs), _p(sn), B, T, H, D, pos0,
                                         int(bool(inverse)), _dt(x), current_stream()))
    return y


def make_rope_tables(seq_len, head_dim, base=1024.0, device="cuda"):
    cs = torch.empty((seq_len, head_dim // 4), dtype=torch.float32, device=device)
    sn = torch.empty_like(cs)
    _lib.check(_lib.lib().ann_op_rope_tables(_p(cs), _p(sn), seq_len, head_dim, float(base), current_stream()))
    return cs, sn


def rms(x, eps=1e-6):
    x = _gpu(x)
    y = torch.empty_like(x)
    dim = x.shape[-1]
    _lib.check(_lib.lib().ann_op_rms_norm(_p(x), _p(y), x.numel() // dim, dim, float(eps),
                                          _dt(x), current_stream()))
    return y


def _table(x, d):
    """cs or sn as the kernel reads it: fp32, contiguous."""
    if not isinstance(x, torch.Tensor) or x.get_device() != d:
        raise ValueError("the tables must be GPU tensors on the rows' device")
    if x.dim() != 2:
        raise ValueError("the tables must be (rows, D/4)")
    if x.dtype is not torch.float32 or not x.is_contiguous():
        x = x.float().contiguous()
    return x


def _qk_struct(q, k, cs, sn, pos, eps, gq=None, gk=None):
    """AnnQkRows of (B, T, H, D) rows, its outputs, the device, and what has to
    outlive the call."""
    rows = (q, k) if gq is None else (q, k, gq, gk)
    d = q.get_device() if isinstance(q, torch.Tensor) else -1
    copied = None
    for i, x in enumerate(rows):
        if not isinstance(x, torch.Tensor) or x.get_device() != d or d < 0:
            raise ValueError("expected GPU tensors on one device")
        if x.dim() != 4:
            raise ValueError("rows must be (B, T, H, D)")
        if x.dtype is not q.dtype:
            raise TypeError(f"dtypes {q.dtype} and {x.dtype} differ")
        if x.stride(3) != 1:
            copied = copied or list(rows)
            copied[i] = x.contiguous()
    if copied:
        rows = copied
        q, k = rows[:2]
    dt = _dt(q)
    B, T, Hq, D = q.shape
    Bk, Tk, Hk, Dk = k.shape
    if Bk != B or Tk != T or Dk != D:
        raise ValueError(f"k {tuple(k.shape)} must be (B, T, Hk, D) of q {tuple(q.shape)}")
    cs, sn = _table(cs, d), _table(sn, d)
    n = cs.shape[0]
    if D % 4 or cs.shape[1] != D // 4 or sn.shape != cs.shape:
        raise ValueError("D must be a multiple of 4 and the tables (rows, D/4)")
    at, each, pos0 = 0, 0, 0
    if isinstance(pos, torch.Tensor):
        if pos.dtype is not torch.int32 or tuple(pos.shape) not in ((B,), (B, T)):
            raise ValueError("pos must be a number or int32 of shape (B,) or (B, T)")
        if pos.get_device() != d:
            raise ValueError("pos must be on the rows' device")
        pos = pos.contiguous()
        at, each = pos.data_ptr(), int(pos.dim() == 2)
    else:
        pos0 = int(pos)
        if B and T and (pos0 < 0 or pos0 + T > n):
            raise ValueError("tables must be (>= pos + T, D/4)")
    g = (0, 0, 0, 0, 0, 0)
    gp = (0, 0)
    if gq is not None:
        gq, gk = rows[2:]
        if gq.shape != q.shape or gk.shape != k.shape:
            raise ValueError(f"gradients {tuple(gq.shape)}, {tuple(gk.shape)} must match "
                             f"{tuple(q.shape)}, {tuple(k.shape)}")
        g = (*gq.stride()[:3], *gk.stride()[:3])
        gp = (gq.data_ptr(), gk.data_ptr())
    qo = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    ko = torch.empty(k.shape, dtype=q.dtype, device=q.device)
    a = _lib.AnnQkRows.from_values(
        q.data_ptr(), k.data_ptr(), 0, *gp, qo.data_ptr(), ko.data_ptr(), *q.stride()[:3],
        *k.stride()[:3], 0, 0, 0, *g, cs.data_ptr(), sn.data_ptr(), at, each, pos0, n, B, T, Hq, Hk,
        D, dt, eps)
    return a, d, qo, ko, (rows, cs, sn, pos)


def _qk_norm_rope(q, k, cs, sn, pos, eps):
    a, d, qo, ko, keep = _qk_struct(q, k, cs, sn, pos, eps)
    _lib.check(on_device(d, _lib.lib().ann_op_qk_norm_rope, a))
    return qo, ko


class _QkNormRope(torch.autograd.Function):
    """``qk_norm_rope`` of rows that require a gradient."""

    @staticmethod
    def forward(ctx, q, k, cs, sn, pos, eps):
        tensor = isinstance(pos, torch.Tensor)
        ctx.save_for_backward(q, k, cs, sn, pos if tensor else None)
        ctx.pos, ctx.eps = None if tensor else pos, eps
        y = _qk_norm_rope(q, k, cs, sn, pos, eps)
        ctx.mark_non_differentiable(*(x for x, need in zip(y, ctx.needs_input_grad) if not need))
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, gq, gk):
        # captured, an accumulation into leaves that an eager graph holds too would
        # end the process: by hand there is none
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("qk_norm_rope: in a captured backward pass call qk_norm_rope_bwd")
        q, k, cs, sn, pos = ctx.saved_tensors
        d = qk_norm_rope_bwd(gq, gk, q, k, cs, sn, ctx.pos if pos is None else pos, ctx.eps)
        return (*(x if need else None for x, need in zip(d, ctx.needs_input_grad)), None, None, None, None)


def qk_norm_rope(q, k, cs, sn, pos=0, eps=1e-6):
    """Queries (B, T, Hq, D) and keys (B, T, Hk, D) as the attention takes them:
    each head's row over sqrt(mean(x^2) + eps), its first half rotated as
    ``rope_ht`` does.  -> (q, k), contiguous, in the input dtype.

    One pass, rounded once: a bf16 result is within one rounding of the exact
    one, where ``rope_ht(rms(x))`` rounds twice.  The inputs may be views with
    any strides over batch, token and head (of a fused projection, say).
    ``pos`` is the position of token 0, or an int32 GPU tensor: (B,) one start
    for each batch row, (B, T) one position for each token (a value outside the
    tables takes their nearest row).

    Autograd passes through to ``q`` and ``k`` (once, by ``qk_norm_rope_bwd``; the
    tables get no gradient), but not in a captured backward pass."""
    if torch.is_grad_enabled() and any(isinstance(x, torch.Tensor) and x.requires_grad for x in (q, k)):
        return _QkNormRope.apply(q, k, cs, sn, pos, eps)
    return _qk_norm_rope(q, k, cs, sn, pos, eps)


def _setting(name, value, rows, dtype, d):
    """(address or 0, the number for all rows, what has to outlive the call)."""
    if not isinstance(value, torch.Tensor):
        return 0, value, None
    if value.dtype is not dtype or tuple(value.shape) != (rows,):
        raise ValueError(f"{name} must be a number or {dtype} of shape {(rows,)}, got {value.dtype} "
                         f"{tuple(value.shape)}")
    if value.get_device() != d:
        raise ValueError(f"{name} must be on the logits' device")
    value = value.contiguous()
    return value.data_ptr(), 0, value


def sample_logits(logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, want_logprob=False):
    """One token of each row of ``logits`` (rows, vocabulary; fp32 or bf16, any row
    stride) by the random numbers ``u`` (rows,) fp32 in [0, 1).  -> ids (rows,)
    int32; with ``want_logprob`` also (rows,) fp32, the log of the share with which
    each was drawn.

    Each setting is a number or a GPU tensor (rows,), ``top_k`` int32, the others
    fp32.  In this order: an entry weighs ``exp((x - max) / temperature)``; weights below
    ``min_p`` (and below 2^-40) are dropped; with ``top_k`` in 1 .. vocabulary - 1 every
    entry below the k-th largest is; with ``top_p`` < 1 all but the largest whose
    weights come to ``top_p`` of what is left.  Equal entries stay or go together.  The token is the
    first index at which the running sum of the weights left passes ``u`` of it.
    Temperature 0 (in a tensor: not above 0) takes the lowest index of the largest
    entry.  A NaN is never drawn; a row of -inf gives -1 and -inf.

    Weights are formed in 64 bits and added exactly, so the same call gives the same tokens.
    Autograd does not see this call."""
    if not (isinstance(logits, torch.Tensor) and logits.is_cuda):
        raise ValueError("expected a GPU tensor")
    if logits.dim() != 2:
        raise ValueError(f"logits must be (rows, vocabulary), got {tuple(logits.shape)}")
    dt, d, device = _dt(logits), logits.get_device(), logits.device
    rows, cols = logits.shape
    if cols > 1 and logits.stride(1) != 1:
        logits = logits.contiguous()
    if not isinstance(u, torch.Tensor):
        raise ValueError("u must be a GPU tensor")
    up, _, u = _setting("u", u, rows, torch.float32, d)
    t, t_all, t_keep = _setting("temperature", temperature, rows, torch.float32, d)
    k, k_all, k_keep = _setting("top_k", top_k, rows, torch.int32, d)
    p, p_all, p_keep = _setting("top_p", top_p, rows, torch.float32, d)
    m, m_all, m_keep = _setting("min_p", min_p, rows, torch.float32, d)
    k_all = min(max(int(k_all), -1), (1 << 31) - 1)
    ids = torch.empty((rows,), dtype=torch.int32, device=device)
    logprob = torch.empty((rows,), dtype=torch.float32, device=device) if want_logprob else None
    a = _lib.AnnLogitRows.from_values(logits.data_ptr(), logits.stride(0), up, t, k, p, m, t_all, k_all,
                                      p_all, m_all, rows, cols, dt, ids.data_ptr(),
                                      logprob.data_ptr() if want_logprob else 0)
    _lib.check(on_device(d, _lib.lib().ann_op_sample_logits, a))
    return (ids, logprob) if want_logprob else ids


def qk_norm_rope_bwd(gq, gk, q, k, cs, sn, pos=0, eps=1e-6):
    """Gradients of ``qk_norm_rope``'s inputs from those of its outputs -> (dq, dk).
    ``q`` and ``k`` are its inputs.  Autograd does not see this call."""
    a, d, qo, ko, keep = _qk_struct(q, k, cs, sn, pos, eps, gq, gk)
    _lib.check(on_device(d, _lib.lib().ann_op_qk_norm_rope_bwd, a))
    return qo, ko
